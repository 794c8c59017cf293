"""b200_op_route and b200_op_gemm_experts against their definitions; an encoder layer of the operators together."""
import ctypes

import numpy as np
import pytest

from lc0_b200 import _lib
from oracle import oracle
from test_gpu_int8 import DT, EPS, activated, quantized, rows

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


# ---- router -----------------------------------------------------------------------------------------------------
def workspace(size_of, d):
    need = ctypes.c_size_t()
    _lib.check(size_of(ctypes.byref(d), ctypes.byref(need)))
    work = torch.full((need.value + 64,), 255, dtype=torch.uint8, device="cuda")  # NaN in every type
    d.workspace, d.workspace_bytes = work.data_ptr(), need.value
    return work


class Route:
    def __init__(self, lib, logits, top_k, renormalise=False, ids=None, experts=None, weights=True):
        n, e = (logits.shape[0], logits.shape[1]) if logits is not None else (ids.shape[0], experts)
        self.lib, self.logits, self.top_k, self.renormalise, self.e, self.n = lib, logits, top_k, renormalise, e, n
        self.ids = ids if ids is not None else torch.full((n, top_k), -7, dtype=torch.int32, device="cuda")
        self.weights = torch.full((n, top_k), NAN, device="cuda") if weights and logits is not None else None
        self.order, self.offsets = (torch.full((s,), -7, dtype=torch.int32, device="cuda") for s in (n * top_k, e + 1))
        self.d = _lib.RouteDesc(logits=None if logits is None else logits.data_ptr(), ld=0 if logits is None else logits.stride(0), rows=n, n_experts=e, top_k=top_k,
                                precision=0 if logits is None else {v: k for k, v in DT.items()}[logits.dtype], renormalise=int(renormalise),
                                ids=self.ids.data_ptr(), weights=None if self.weights is None else self.weights.data_ptr(), order=self.order.data_ptr(),
                                offsets=self.offsets.data_ptr())
        self.work = workspace(lib.b200_op_route_workspace, self.d)

    def call(self, stream=None):
        _lib.check(self.lib.b200_op_route(ctypes.byref(self.d), stream))

    def run(self, stream=None):
        torch.cuda.synchronize()
        self.call(stream)
        torch.cuda.synchronize()
        assert (self.work[-64:] == 255).all()
        return self

    def check(self):
        if self.logits is not None:
            l = self.logits.double().cpu().numpy()
            l = np.where(np.isnan(l), -INF, l)
            want = np.argsort(-l, axis=1, kind="stable")[:, :self.top_k]
            chosen = np.take_along_axis(l, want, axis=1)
            want = np.where(chosen > -INF, want, -1)
            assert np.array_equal(self.ids.cpu().numpy(), want)
            if self.weights is not None:
                top = l.max(axis=1, keepdims=True)
                with np.errstate(invalid="ignore"):
                    w = np.where(l == top, 1.0, np.where(top == INF, 0.0, np.exp(l - top)))
                w = np.where(l > -INF, w, 0.0)
                c = np.where(want >= 0, np.take_along_axis(w, np.maximum(want, 0), axis=1), 0.0)
                total = (c if self.renormalise else w).sum(axis=1, keepdims=True)
                w = np.divide(c, total, out=np.zeros_like(c), where=total > 0)
                # expf: two steps, and half a step of its argument, which is at most 104 where the result counts; sums of at most 8 + 5 steps
                assert np.abs(self.weights.double().cpu().numpy() - w).max() <= 1e-37 + (2 * 104 + 40) * 2.0 ** -24 * 1.0
                assert (np.abs(self.weights.double().cpu().numpy() - w) <= 1e-37 + 300 * 2.0 ** -24 * w).all()
        flat = self.ids.reshape(-1).cpu().numpy()
        placed = np.flatnonzero((flat >= 0) & (flat < self.e))
        order = placed[np.argsort(flat[placed], kind="stable")]
        assert np.array_equal(self.order[:order.size].cpu().numpy(), order)
        assert (self.order[order.size:] == -7).all()
        assert np.array_equal(self.offsets.cpu().numpy(), np.concatenate([[0], np.cumsum(np.bincount(flat[placed], minlength=self.e))]))


@gpu
@pytest.mark.parametrize("prec", [0, 1, 2])
@pytest.mark.parametrize("n,e,top_k", [(1, 1, 1), (1, 8, 8), (3, 2, 1), (37, 5, 2), (64, 8, 1), (100, 9, 4), (1536, 16, 2), (1000, 33, 3), (777, 64, 16), (5, 256, 16),
                                       (4100, 100, 8), (65536, 64, 4), (30000, 256, 2), (100003, 7, 2), (2048, 128, 6)])
def test_route(lib, prec, n, e, top_k):
    g = torch.Generator(device="cuda").manual_seed(n + e)
    l = torch.randn(n, e, device="cuda", generator=g) * 1.5 + 2 * torch.randn(e, device="cuda", generator=g)
    Route(lib, l.to(DT[prec]), top_k, renormalise=(n + prec) % 2 == 1).run().check()
    Route(lib, rows(n, e, 3, l.to(DT[prec]), NAN, 1), top_k, renormalise=(n + prec) % 2 == 0).run().check()


@gpu
@pytest.mark.parametrize("e", [3, 16, 50, 256])
@pytest.mark.parametrize("renormalise", [False, True])
def test_route_ties_and_what_is_no_number(lib, e, renormalise):
    """Equal logits by index, zeros of both signs among them; rows of NaN and -infinity alone; infinities; the ends of the type; far logits."""
    for prec in (0, 1, 2):
        t = DT[prec]
        l = torch.randint(-2, 3, (200, e), device="cuda").to(t)
        l[1::5] *= -0.0
        l[0] = 1.0
        l[2], l[3] = NAN, -INF
        l[4, ::2] = -INF
        l[5, ::3], l[6, 1:] = INF, NAN
        l[7] = torch.finfo(t).min
        l[8], l[8, 2] = torch.finfo(t).min, torch.finfo(t).max
        l[9, :2] = torch.tensor([-INF, NAN])
        l[10] = -90.0 * torch.arange(e, device="cuda")
        Route(lib, l, min(e, 4), renormalise).run().check()
        Route(lib, l, min(e, 16), renormalise, weights=False).run().check()


@gpu
@pytest.mark.parametrize("rows", [300, 20000])
@pytest.mark.parametrize("experts", [32, 64, 128, 256])
def test_float_weights_are_of_rounded_exponentials(lib, rows, experts):
    """fp32 logits: the softmax's denominator takes expf, off by two steps at most as CUDA documents it, so one of five numbers around the rounded
    exponential.  One logit of 0 beside equal ones x: eight of a lane are added in order, then the lanes in pairs, so with each of the five the weight
    1 / sum is one number."""
    f = np.float32
    x = np.random.default_rng(experts).uniform(-7, -0.5, rows).astype(f)
    l = np.repeat(x[:, None], experts, axis=1)
    first = np.arange(rows) % experts
    l[np.arange(rows), first] = 0
    r = Route(lib, torch.from_numpy(l).cuda(), 1).run()
    r.check()
    best = np.exp(x.astype(np.float64)).astype(f)
    sums = []
    for step in range(-2, 3):
        e = (best.view(np.int32) + np.int32(step)).view(f)
        terms = np.repeat(e[:, None], experts, axis=1)
        terms[np.arange(rows), first] = 1
        lanes = terms.reshape(rows, experts // 8, 8)
        total = np.zeros((rows, experts // 8), f)
        for i in range(8):
            total = total + lanes[:, :, i]
        while total.shape[1] > 1:
            half = total.shape[1] // 2
            total = total[:, :half] + total[:, half:]
        sums.append(f(1) / total[:, 0])
    assert total.dtype == f
    got = r.weights.cpu().numpy()[:, 0]
    assert (got <= np.maximum.reduce(sums)).all() and (got >= np.minimum.reduce(sums)).all()


@gpu
@pytest.mark.parametrize("n,e,top_k", [(1, 1, 1), (24, 8, 1), (333, 12, 1), (70000, 256, 3), (5000, 1, 2), (100, 5, 16)])
def test_route_of_given_ids(lib, n, e, top_k):
    ids = torch.randint(-2, e + 2, (n, top_k), dtype=torch.int32, device="cuda")
    ids[n // 3:n // 2] = 0
    before = ids.clone()
    Route(lib, None, top_k, ids=ids, experts=e).run().check()
    assert torch.equal(ids, before)
    ids.fill_(-1)
    Route(lib, None, top_k, ids=ids, experts=e).run().check()


@gpu
def test_route_without_rows(lib):
    offsets = torch.full((9,), -7, dtype=torch.int32, device="cuda")
    _lib.check(lib.b200_op_route(ctypes.byref(_lib.RouteDesc(rows=0, n_experts=8, top_k=2, offsets=offsets.data_ptr())), None))
    torch.cuda.synchronize()
    assert not offsets.any()


# ---- products ---------------------------------------------------------------------------------------------------
class Experts:
    """side: up (tokens to slots), down (slots to tokens), head (tokens to tokens) or slots (slots to slots)."""

    def __init__(self, lib, side, requests, N, K, experts, top_k=1, group=1, prec=1, int8=False, f32=False, act=oracle.ACT_NONE, bias=True, weights=None, res=False,
                 ids=None, pads=(0, 0, 0), shift=0, seed=0, in_place=False):
        g = torch.Generator(device="cuda").manual_seed(seed + requests + 3 * N + 7 * K + experts)
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
        whole = lambda *s: torch.randint(-127, 128, s, device="cuda", generator=g).to(torch.int8)
        t, M = DT[prec], requests * group
        self.side, self.requests, self.M, self.N, self.K, self.e, self.top_k, self.group = side, requests, M, N, K, experts, top_k, group
        self.prec, self.int8, self.f32, self.act, self.lib = prec, int8, f32 or prec == 0, act, lib
        if ids is None:  # few popular experts, some choices without one
            ids = (rnd(requests, experts) + 1.5 * rnd(experts)).topk(top_k, dim=1).indices
            ids = torch.where(torch.rand(requests, top_k, device="cuda", generator=g) < 0.1, -1, ids)
        self.ids = torch.as_tensor(ids, dtype=torch.int32, device="cuda").reshape(requests, top_k).contiguous()
        self.by_slot, self.from_slots = side in ("up", "slots"), side in ("down", "slots")
        n_x = M * top_k if self.from_slots else M
        self.x = rows(n_x, K, pads[0], whole(n_x, K) if int8 else rnd(n_x, K).to(t), 99 if int8 else NAN, shift)
        w = whole(experts * N, K) if int8 else (rnd(experts * N, K) * K ** -0.5).to(t)
        self.w = rows(experts * N, K, pads[1], w, 99 if int8 else NAN, shift)
        self.sx, self.sw = (0.5 + torch.rand(n_x, device="cuda", generator=g)) / 73, (0.5 + torch.rand(experts, N, device="cuda", generator=g)) / 73 * K ** -0.5
        self.bias = rnd(experts, N) if bias else None
        out_t = torch.float32 if self.f32 else t
        n_c = M * top_k if self.by_slot else M
        self.out = rows(n_c, N, pads[2], torch.full((n_c, N), 55.0, dtype=out_t, device="cuda"), 77.0, shift)
        self.res = rows(M, N, pads[2], rnd(M, N).to(out_t), NAN, shift) if res else None
        if in_place:
            self.out.copy_(self.res)
        self.in_place = in_place
        self.weights = torch.rand(requests, top_k, device="cuda", generator=g) if (not self.by_slot if weights is None else weights) else None
        key = torch.where((self.ids < 0) | (self.ids >= experts), experts, self.ids.long()).reshape(-1)
        self.order = torch.argsort(key, stable=True).int()
        self.offsets = torch.cat([key.new_zeros(1), torch.bincount(key, minlength=experts + 1)[:experts].cumsum(0)]).int()
        self.slots = int(self.offsets[-1]) * group
        self.order[self.slots // group:] = -7  # what lies there is nobody's
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        p = lambda v: None if v is None else v.data_ptr()
        self.d = _lib.ExpertsDesc(X=p(self.x), W=p(self.w), bias=p(self.bias), C=p(self.out), M=M, N=N, K=K, ldx=self.x.stride(0), ldw=self.w.stride(0),
                                  ldc=self.out.stride(0), activation=act, precision=prec, out_f32=int(f32), int8=int(int8), x_scales=p(self.sx) if int8 else None,
                                  w_scales=p(self.sw) if int8 else None, n_experts=experts, top_k=top_k, group=group, ids=p(self.ids), order=p(self.order),
                                  offsets=p(self.offsets), x_by_slot=int(self.from_slots), c_by_slot=int(self.by_slot), weights=p(self.weights),
                                  res=p(self.out if in_place else self.res), ldres=self.out.stride(0), status=p(self.status))
        self.work = workspace(lib.b200_op_gemm_experts_workspace, self.d)

    def run(self, stream=None):
        torch.cuda.synchronize()
        _lib.check(self.lib.b200_op_gemm_experts(ctypes.byref(self.d), stream))
        torch.cuda.synchronize()
        assert self.status.item() == 0 and (self.work[-64:] == 255).all()
        return self

    def want(self):
        """The result, what it may be off by ahead of its rounding, and which rows are written.  int8 as in the plain product; else sums of K
        products in fp32, K rounded additions at most."""
        n_c = self.M * self.top_k if self.by_slot else self.M
        out, err = torch.zeros(n_c, self.N, dtype=torch.float64, device="cuda"), torch.zeros(n_c, self.N, dtype=torch.float64, device="cuda")
        written = torch.zeros(n_c, dtype=torch.bool, device="cuda")
        if self.res is not None:
            out += self.res.double()
        at, order = self.offsets.tolist(), self.order.long()
        inside = torch.arange(self.group, device="cuda")
        for e in range(self.e):
            if at[e] == at[e + 1]:
                continue
            choice = order[at[e]:at[e + 1]]
            slot = torch.arange(at[e] * self.group, at[e + 1] * self.group, device="cuda")
            token = ((choice // self.top_k)[:, None] * self.group + inside).view(-1)
            src = slot if self.from_slots else token
            x, w = self.x[src].double(), self.w[e * self.N:(e + 1) * self.N].double()
            if self.int8:
                y = (x @ w.T) * (self.sx[src].double()[:, None] * self.sw[e].double())
                mag, steps = y.abs(), 4
            else:
                y, mag, steps = x @ w.T, x.abs() @ w.abs().T, self.K + 2
            if self.bias is not None:
                y, mag = y + self.bias[e].double(), mag + self.bias[e].double().abs()
            v, off = activated(y, steps * 2.0 ** -24 * mag, self.act, self.prec != 0 and not self.f32 and (self.by_slot or self.top_k == 1))
            if self.weights is not None:
                wt = self.weights.view(-1)[choice].double().repeat_interleave(self.group)[:, None]
                v, off = v * wt, (off + 2.0 ** -24 * v.abs()) * wt
            dst = slot if self.by_slot else token
            out.index_add_(0, dst, v)
            err.index_add_(0, dst, off + 2.0 ** -24 * (v.abs() + out[dst].abs()) * (0 if self.by_slot else 1))
            written[dst] = True
        return out, err, written

    def check(self):
        want, err, written = self.want()
        half = EPS[0] if self.f32 else EPS[self.prec]
        allowed = half * (want.abs() + err) + err + (2.0 ** -25 if self.prec == 1 and not self.f32 else 1e-37)
        off = ((self.out.double() - want).abs() / allowed)[written]
        if off.numel():
            assert off.max().item() <= 1, off.max().item()  # NaN fails
        left = self.out[~written]
        assert torch.equal(left, self.res[~written] if self.in_place else torch.full_like(left, 55.0))
        n = self.out.shape[0]
        if self.out.stride(0) > self.N and n > 1:
            gap = torch.as_strided(self.out, (n - 1, self.out.stride(0) - self.N), (self.out.stride(0), 1), self.out.storage_offset() + self.N)
            assert (gap == 77).all()


@gpu
@pytest.mark.parametrize("prec,int8", [(1, False), (2, False), (1, True), (2, True), (0, True)])
@pytest.mark.parametrize("side", ["up", "down", "head"])
@pytest.mark.parametrize("requests,N,K,experts,top_k,group", [
    (1, 1, 1, 1, 1, 1), (1, 16, 32, 8, 2, 1), (5, 130, 45, 3, 1, 1), (37, 264, 128, 12, 1, 1), (100, 64, 64, 40, 3, 1), (333, 1858, 256, 12, 1, 1), (24, 512, 256, 8, 1, 64),
    (3, 96, 144, 2, 1, 64), (700, 256, 512, 5, 2, 1), (1500, 520, 320, 16, 4, 1), (4096, 384, 256, 16, 2, 1), (64, 256, 384, 6, 2, 64), (20, 136, 1040, 4, 1, 5),
    (2000, 256, 128, 1, 1, 1), (3000, 1024, 1536, 4, 1, 1), (300, 64, 64, 256, 8, 1)])
def test_products(lib, prec, int8, side, requests, N, K, experts, top_k, group):
    act = [oracle.ACT_NONE, oracle.ACT_MISH, oracle.ACT_RELU_2, oracle.ACT_SWISH][(requests + prec) % 4]
    Experts(lib, side, requests, N, K, experts, top_k, group, prec, int8, act=act, res=side != "up" and (N + prec) % 2 == 0).run().check()


@gpu
@pytest.mark.parametrize("side,top_k", [("head", 1), ("up", 1), ("up", 2), ("down", 2), ("head", 2)])
@pytest.mark.parametrize("requests,N,K", [(1, 1858, 512), (333, 1858, 1024), (2500, 256, 512), (5000, 512, 128)])
@pytest.mark.parametrize("prec,int8", [(1, False), (2, False), (2, True)])
def test_float_results(lib, side, top_k, requests, N, K, prec, int8):
    c = Experts(lib, side, requests, N, K, 6, top_k, 1, prec, int8, f32=True, res=side == "head", act=oracle.ACT_MISH if top_k == 2 else oracle.ACT_NONE).run()
    c.check()
    if not int8 and c.act == oracle.ACT_NONE and c.res is None:  # as exact as a plain product in fp32, in the root mean square
        want, _, written = c.want()
        plain, at = torch.zeros_like(c.out), c.offsets.tolist()
        for e in range(c.e):
            choice = c.order[at[e]:at[e + 1]].long()
            y = c.x[choice // top_k].float() @ c.w[e * N:(e + 1) * N].float().T + c.bias[e]
            plain[at[e]:at[e + 1]] = y
        if side == "up" and requests > 1:
            rms = lambda v: (v.double() - want)[written].square().mean().sqrt().item()
            assert rms(c.out) <= 1.5 * rms(plain) + 2.0 ** -26


@gpu
@pytest.mark.parametrize("pads,shift", [((8, 16, 8), 0), ((5, 0, 0), 0), ((0, 3, 1), 0), ((0, 0, 3), 1), ((16, 16, 8), 16)])
@pytest.mark.parametrize("side,top_k", [("up", 2), ("down", 2), ("head", 1)])
@pytest.mark.parametrize("int8", [False, True])
def test_strides(lib, pads, shift, side, top_k, int8):
    Experts(lib, side, 300, 200, 256, 5, top_k, 1, 2, int8, pads=pads, shift=shift, res=side != "up").run().check()
    Experts(lib, side, 7, 50, 176, 3, top_k, 64, 1, int8, pads=pads, shift=shift, res=side != "up").run().check()


@gpu
@pytest.mark.parametrize("side", ["up", "down", "head"])
@pytest.mark.parametrize("top_k,group", [(1, 1), (2, 1), (1, 64)])
@pytest.mark.parametrize("int8", [False, True])
def test_lopsided_choices(lib, side, top_k, group, int8):
    """All requests with one expert, none with any, one row each, the last expert alone, ids far outside."""
    n, e = 300 if group == 1 else 9, 20
    cases = [torch.full((n, top_k), 3), torch.full((n, top_k), -1), torch.arange(n * top_k).view(n, top_k) % e, torch.full((n, top_k), e - 1),
             torch.where(torch.arange(n * top_k).view(n, top_k) % 7 == 0, 2 ** 31 - 1, torch.arange(n * top_k).view(n, top_k) % e)]
    for i, ids in enumerate(cases):
        Experts(lib, side, n, 136, 256, e, top_k, group, 1, int8, ids=ids, seed=i).run().check()


@gpu
@pytest.mark.parametrize("prec,requests,N,top_k", [(1, 300, 264, 1), (2, 5000, 512, 2), (1, 40, 50, 2)])
def test_residual_in_place_and_no_weights(lib, prec, requests, N, top_k):
    Experts(lib, "down", requests, N, 256, 8, top_k, 1, prec, res=True, in_place=True).run().check()
    Experts(lib, "head", requests, N, 256, 8, top_k, 1, prec, res=True, weights=False, bias=False).run().check()


@gpu
@pytest.mark.parametrize("requests", [20, 700])
def test_weights_beyond_32_bits(lib, requests):
    """The last expert's weights lie more than 2^32 behind the first's."""
    e, N, K = 70, 8192, 8192
    c = Experts(lib, "head", requests, N, 64, 1, 1, 1, 1, int8=True, ids=torch.zeros(requests, 1))
    w = torch.zeros(e, N, K, dtype=torch.int8, device="cuda")
    w[-1].random_(-127, 128)
    x = torch.randint(-127, 128, (requests, K), device="cuda").to(torch.int8)
    sw, bias = torch.ones(e, N, device="cuda"), torch.zeros(e, N, device="cuda")
    sw[-1], bias[-1] = c.sw[0] / 10, c.bias[0]
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    offsets[-1] = requests
    c.d.X, c.d.W, c.d.ldx, c.d.ldw, c.d.K, c.d.n_experts = x.data_ptr(), w.data_ptr(), K, K, K, e
    c.d.w_scales, c.d.bias, c.d.offsets = sw.data_ptr(), bias.data_ptr(), offsets.data_ptr()
    work = workspace(lib.b200_op_gemm_experts_workspace, c.d)
    c.run()
    c.x, c.w, c.sw, c.bias, c.K = x, w[-1], sw[-1:], bias[-1:], K
    c.check()
    assert (work[-64:] == 255).all()


@gpu
@pytest.mark.parametrize("requests,N,K,experts,top_k,group", [(50, 264, 128, 6, 2, 1), (2000, 512, 320, 4, 2, 1), (40, 300, 192, 3, 1, 64), (9, 70, 33, 3, 2, 1)])
@pytest.mark.parametrize("int8", [False, True])
def test_from_slots_to_slots(lib, requests, N, K, experts, top_k, group, int8):
    Experts(lib, "slots", requests, N, K, experts, top_k, group, 2, int8, act=oracle.ACT_SWISH).run().check()


@gpu
@pytest.mark.parametrize("requests,N,K,experts,top_k", [(3000, 512, 256, 4, 2), (300, 264, 128, 4, 2), (70, 136, 64, 40, 1)])
def test_calls_at_once(lib, requests, N, K, experts, top_k):
    """The same product on four streams at once, a workspace and outputs each, again and again."""
    calls = [Experts(lib, "down", requests, N, K, experts, top_k, 1, 1 + i % 2, seed=i, res=True) for i in range(4)]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(8):
        for c, st in zip(calls, streams):
            _lib.check(lib.b200_op_gemm_experts(ctypes.byref(c.d), st.cuda_stream))
    torch.cuda.synchronize()
    for c in calls:
        assert c.status.item() == 0
        c.check()


@gpu
@pytest.mark.parametrize("int8", [False, True])
def test_what_is_not_finite_stays_in_its_rows(lib, int8):
    """Another expert's weights and another request's rows, NaN or infinite, reach nobody else."""
    for requests in (60, 900):
        c = Experts(lib, "head", requests, 136, 256, 4, 1, 1, 1, int8, ids=torch.arange(requests)[:, None] % 4)
        if int8:
            c.sx[5], c.sw[2] = NAN, INF
        else:
            c.x[5], c.w[2 * 136:3 * 136] = NAN, INF
        c.run()
        bad = (torch.arange(requests, device="cuda") % 4 == 2) | (torch.arange(requests, device="cuda") == 5)
        assert (~c.out.isfinite()).any(dim=1)[5] and c.out[~bad].isfinite().all()


@gpu
def test_bad_lists_stay_inside(lib):
    """Offsets and places outside the slots name no rows: nothing outside the outputs is written, and the rows that are named are right."""
    c = Experts(lib, "head", 200, 72, 64, 4, 1, 1, 1, ids=torch.arange(200)[:, None] % 4, pads=(0, 0, 8))
    c.order[10], c.order[60] = 200, -5
    c.offsets[4] = 10 ** 9
    c.run()
    lost = torch.zeros(200, dtype=torch.bool, device="cuda")
    lost[[40, 41]] = True  # places 10 of expert 0 (request 40) and 10 of expert 1 (request 41)
    want, err, _ = Experts(lib, "head", 200, 72, 64, 4, 1, 1, 1, ids=torch.arange(200)[:, None] % 4, pads=(0, 0, 8)).want()
    assert (c.out[lost] == 55).all()
    assert ((c.out.double() - want).abs() <= EPS[1] * want.abs() + 2 * err + 2.0 ** -25)[~lost].all()
    gap = torch.as_strided(c.out, (199, 8), (80, 1), 72)
    assert (gap == 77).all()


@gpu
def test_rows_do_not_depend_on_their_neighbours(lib):
    """A request's row alone with its expert and among all others."""
    whole = Experts(lib, "head", 3000, 264, 512, 6, 1, 1, 2, act=oracle.ACT_MISH, ids=torch.arange(3000)[:, None] % 6, seed=3).run()
    ids = torch.full((3000, 1), -1)
    ids[::100] = (torch.arange(3000) % 6)[::100, None]
    few = Experts(lib, "head", 3000, 264, 512, 6, 1, 1, 2, act=oracle.ACT_MISH, ids=ids, seed=3).run()
    assert ((few.out[::100].float() - whole.out[::100].float()).abs() <= 2.0 ** -8 * whole.out[::100].float().abs() + 1e-6).all()


@gpu
def test_two_graphs_and_a_stream(lib):
    """Router and products captured once, replayed with other logits, two graphs at once on two streams."""
    n, e, top_k, N, K = 800, 8, 2, 256, 192
    made, graphs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for i, st in enumerate(streams):
        logits = torch.randn(n, e, device="cuda")
        r = Route(lib, logits, top_k, True)
        up = Experts(lib, "up", n, N, K, e, top_k, 1, 2, seed=i, act=oracle.ACT_MISH)
        down = Experts(lib, "down", n, K, N, e, top_k, 1, 2, seed=i + 5, res=True)
        for c in (up, down):
            c.d.order, c.d.offsets, c.d.ids = r.order.data_ptr(), r.offsets.data_ptr(), r.ids.data_ptr()
        down.d.weights, down.d.X, down.d.ldx = r.weights.data_ptr(), up.out.data_ptr(), up.out.stride(0)
        torch.cuda.synchronize()

        def calls():
            s = torch.cuda.current_stream().cuda_stream
            r.call(s)
            for c in (up, down):
                _lib.check(lib.b200_op_gemm_experts(ctypes.byref(c.d), s))

        with torch.cuda.stream(st):
            calls()
        st.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            calls()
        graphs.append(graph)
        made.append((r, up, down))
    for turn in range(3):
        for r, up, down in made:
            r.logits.normal_()
            up.x.normal_()
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for r, up, down in made:
            r.check()
            for c in (up, down):
                c.order, c.offsets, c.ids = r.order, r.offsets, r.ids
                c.x, c.weights = (up.out, r.weights) if c is down else (c.x, None)
                c.check()


@gpu
@pytest.mark.parametrize("n", [1, 24, 200])
def test_an_encoder_layer(lib, n):
    """The operators as an encoder layer uses them, behind and before what was there: Q, K and V by an 8-bit product, norms and rotation of Q and
    K, b200_op_attention, the projection in 8 bits with the residual, and a layer of experts that each position, or each token, chooses."""
    g = torch.Generator(device="cuda").manual_seed(n)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    C, H, depth, E, F, T = 256, 8, 32, 4, 320, n * 64
    h = torch.float16
    st = torch.cuda.Stream()
    s = st.cuda_stream
    empty = lambda *shape, dtype=h: torch.empty(*shape, dtype=dtype, device="cuda")
    ptr = lambda v: v.data_ptr()
    x = rnd(T, C).to(h)
    w_qkv, w_out = quantized(rnd(3 * C, C) * C ** -0.5), quantized(rnd(C, C) * C ** -0.5)
    w1, w2 = (rnd(E, F, C) * C ** -0.5).to(h), (rnd(E, C, F) * F ** -0.5).to(h)
    b1, b2 = rnd(E, F) * 0.1, rnd(E, C) * 0.1
    gq, gk = 1 + 0.1 * rnd(depth), 1 + 0.1 * rnd(depth)
    angle = (torch.arange(64, device="cuda")[:, None] * 8.0 ** -torch.arange(depth // 2, device="cuda")[None]).double()
    table = torch.stack([angle.cos(), angle.sin()], dim=2).float().contiguous()
    wr = (rnd(E, C) * C ** -0.5).to(h)

    def layer8(inp, w, out, res=None):
        m, k = inp.shape
        q, sx = empty(m, k, dtype=torch.int8), empty(m, dtype=torch.float32)
        held.extend([q, sx])
        _lib.check(lib.b200_op_quantize_rows(ptr(inp), 0, m, k, 1, ptr(q), 0, ptr(sx), s))
        d = _lib.GemmInt8Desc(X=ptr(q), x_scales=ptr(sx), W=ptr(w[0]), w_scales=ptr(w[1]), C=ptr(out), M=m, N=w[0].shape[0], K=k, activation=oracle.ACT_NONE,
                              precision=1, alpha=1.0, res=None if res is None else ptr(res), status=ptr(status))
        _lib.check(lib.b200_op_gemm_int8(ctypes.byref(d), s))

    def exact8(inp, w):
        q, sx = quantized(inp)
        return (q.double() * sx.double()[:, None]) @ (w[0].double() * w[1].double()[:, None]).T

    for per_token in (False, True):
        held, status = [], torch.zeros(1, dtype=torch.int32, device="cuda")
        qkv, att, y, out = empty(T, 3 * C), empty(T, C), empty(T, C), torch.zeros(T, C, dtype=h, device="cuda")
        top_k, group = (2, 1) if per_token else (1, 64)
        requests = T // group
        logits, mid = empty(requests, E, dtype=torch.float32), empty(T * top_k, F)
        torch.cuda.synchronize()
        layer8(x, w_qkv, qkv)
        q, k, v = qkv[:, :C], qkv[:, C:2 * C], qkv[:, 2 * C:]
        _lib.check(lib.b200_op_qk_norm_rotate(ctypes.byref(_lib.QkNormDesc(
            q=ptr(q), k=ptr(k), ldq=3 * C, ldk=3 * C, q_out=ptr(q), k_out=ptr(k), ldq_out=3 * C, ldk_out=3 * C, rows=T, q_heads=H, k_heads=H, depth=depth, precision=1,
            norm=1, eps=1e-6, gamma_q=ptr(gq), gamma_k=ptr(gk), rotate=depth, table=ptr(table), n_positions=64)), s))
        _lib.check(lib.b200_op_attention(ptr(q), ptr(k), ptr(v), 3 * C, None, ptr(att), C, n, H, depth, 1, 1, s))
        layer8(att, w_out, y, res=x)
        with torch.cuda.stream(st):  # the router's small product
            first = y.float().view(requests, group, C).mean(1)
            torch.matmul(first, wr.float().T, out=logits)
        r = Route(lib, logits, top_k, True)
        st.wait_stream(torch.cuda.current_stream())
        r.call(s)
        up = _lib.ExpertsDesc(X=ptr(y), W=ptr(w1), bias=ptr(b1), C=ptr(mid), M=T, N=F, K=C, activation=oracle.ACT_SWISH, precision=1, n_experts=E, top_k=top_k, group=group,
                              order=ptr(r.order), offsets=ptr(r.offsets), c_by_slot=1, status=ptr(status))
        down = _lib.ExpertsDesc(X=ptr(mid), W=ptr(w2), bias=ptr(b2), C=ptr(out), M=T, N=C, K=F, activation=oracle.ACT_NONE, precision=1, n_experts=E, top_k=top_k,
                                group=group, ids=ptr(r.ids), order=ptr(r.order), offsets=ptr(r.offsets), x_by_slot=1, weights=ptr(r.weights), res=ptr(y), status=ptr(status))
        work = [workspace(lib.b200_op_gemm_experts_workspace, d) for d in (up, down)]
        st.wait_stream(torch.cuda.current_stream())
        for d in (up, down):
            _lib.check(lib.b200_op_gemm_experts(ctypes.byref(d), s))
        torch.cuda.synchronize()
        assert status.item() == 0 and all((w[-64:] == 255).all() for w in work)
        # step by step in 64 bits, each from the values that the step before it left
        def near(got, want, steps):
            # fp16: half a step of the result, and `steps` of the values on the way
            scale = want.abs() + want.square().mean().sqrt()
            assert ((got.double() - want).abs() <= steps * 2.0 ** -11 * scale).all()

        near(qkv[:, 2 * C:], exact8(x, w_qkv)[:, 2 * C:], 2)
        full = exact8(x, w_qkv)

        def turned(v, gamma):
            v = v.view(T, H, depth)
            v = v / torch.sqrt(v.square().mean(2, keepdim=True) + 1e-6) * gamma.double()
            t = table.double().repeat(n, 1, 1)[:, None]
            a, b = v[..., :depth // 2], v[..., depth // 2:]
            return torch.cat([a * t[..., 0] - b * t[..., 1], a * t[..., 1] + b * t[..., 0]], 2).reshape(T, C)

        near(qkv[:, :C], turned(full[:, :C].half().double(), gq), 4)
        near(qkv[:, C:2 * C], turned(full[:, C:2 * C].half().double(), gk), 4)
        heads = lambda v: v.double().reshape(n, 64, H, depth).transpose(1, 2)
        a = torch.softmax(heads(q) @ heads(k).transpose(2, 3) * depth ** -0.5, dim=3) @ heads(v)
        near(att, a.transpose(1, 2).reshape(T, C), 6)
        near(y, exact8(att, w_out) + x.double(), 2)
        r.check()
        choice = r.ids.long().repeat_interleave(group, dim=0)
        slot = torch.empty(requests * top_k, dtype=torch.long, device="cuda")
        slot[r.order.long()] = torch.arange(requests * top_k, device="cuda")
        want = y.double()
        for j in range(top_k):
            for e in range(E):
                t = (choice[:, j] == e).nonzero()[:, 0]
                at = slot[(t // group) * top_k + j] * group + t % group
                z = y[t].double() @ w1[e].double().T + b1[e].double()
                near(mid[at], z * torch.sigmoid(z), 3) if t.numel() else None
                want[t] += r.weights[t // group, j].double()[:, None] * (mid[at].double() @ w2[e].double().T + b2[e].double())
        near(out, want, 2)


def test_route_refusals(lib):
    def call(**kw):
        d = _lib.RouteDesc(logits=256, rows=4, n_experts=8, top_k=2, precision=1, ids=256, weights=256, order=256, offsets=256, workspace=256, workspace_bytes=1 << 30)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.b200_op_route(ctypes.byref(d), None)

    need = ctypes.c_size_t()
    assert lib.b200_op_route(None, None) == _lib.ERR_INVALID
    assert lib.b200_op_route_workspace(None, ctypes.byref(need)) == _lib.ERR_INVALID
    assert lib.b200_op_route_workspace(ctypes.byref(_lib.RouteDesc(rows=4, n_experts=8, top_k=2, precision=1)), None) == _lib.ERR_INVALID
    for kw in (dict(rows=-1), dict(n_experts=0), dict(n_experts=257), dict(top_k=0), dict(top_k=9), dict(n_experts=32, top_k=17), dict(precision=3), dict(ld=7),
               dict(ids=None), dict(order=None), dict(offsets=None), dict(logits=None), dict(logits=257), dict(ids=258), dict(weights=257), dict(order=257),
               dict(offsets=258), dict(workspace=None), dict(workspace=128), dict(workspace_bytes=16), dict(rows=2 ** 30, top_k=8)):
        assert call(**kw) == _lib.ERR_INVALID, kw
        assert b"b200_op_route" in lib.b200_last_error()


def test_products_refusals(lib):
    good = dict(X=256, W=256, C=256, M=64, N=8, K=64, activation=3, precision=1, n_experts=4, top_k=2, group=1, ids=256, order=256, offsets=256, workspace=256,
                workspace_bytes=1 << 30)

    def call(**kw):
        return lib.b200_op_gemm_experts(ctypes.byref(_lib.ExpertsDesc(**dict(good, **kw))), None)

    need = ctypes.c_size_t()
    assert lib.b200_op_gemm_experts(None, None) == _lib.ERR_INVALID
    assert lib.b200_op_gemm_experts_workspace(None, ctypes.byref(need)) == _lib.ERR_INVALID
    assert lib.b200_op_gemm_experts_workspace(ctypes.byref(_lib.ExpertsDesc(**good)), None) == _lib.ERR_INVALID
    assert call(M=0) == _lib.OK
    for kw in (dict(M=-64), dict(N=0), dict(K=0), dict(K=131072), dict(int8=1, x_scales=256, w_scales=256, K=131072), dict(n_experts=0), dict(n_experts=257), dict(top_k=0), dict(top_k=17),
               dict(group=0), dict(group=48), dict(M=2 ** 30), dict(N=2 ** 30), dict(precision=0), dict(precision=3), dict(activation=0), dict(activation=9), dict(ldx=63),
               dict(ldw=63), dict(ldc=7), dict(res=256, ldres=7), dict(c_by_slot=1, weights=256), dict(c_by_slot=1, res=256), dict(X=None), dict(W=None), dict(C=None),
               dict(order=None), dict(offsets=None), dict(ids=None), dict(int8=1), dict(int8=1, x_scales=256), dict(X=257), dict(W=257), dict(C=257), dict(C=258, out_f32=1),
               dict(res=257), dict(bias=258), dict(order=258), dict(offsets=257), dict(weights=258), dict(status=258), dict(res=256, ldres=16), dict(workspace=None),
               dict(workspace=128), dict(workspace_bytes=2047)):
        assert call(**kw) == _lib.ERR_INVALID, kw
        assert b"b200_op_gemm_experts" in lib.b200_last_error()


_CALLS = r"""
import ctypes, sys
from lc0_b200 import _lib
lib, shim = _lib.load(), ctypes.CDLL(sys.argv[1])
need = ctypes.c_size_t()
gemm, route, experts, norm = _lib.GemmInt8Desc(M=-1), _lib.RouteDesc(rows=-1), _lib.ExpertsDesc(M=-1), _lib.QkNormDesc(rows=-1)
ref = ctypes.byref
shim.no_more_memory(1)
codes = [lib.b200_op_quantize_rows(None, 0, -1, 0, 0, None, 0, None, None), lib.b200_op_gemm_int8(ref(gemm), None), lib.b200_op_route(ref(route), None),
         lib.b200_op_route_workspace(ref(route), ref(need)), lib.b200_op_gemm_experts(ref(experts), None), lib.b200_op_gemm_experts_workspace(ref(experts), ref(need)),
         lib.b200_op_qk_norm_rotate(ref(norm), None)]
shim.no_more_memory(0)
print(codes, lib.b200_op_gemm_int8(ref(gemm), None))
"""


def test_without_host_memory(tmp_path):
    """An allocation that fails inside a call (the message of a refusal is one) is an error code, not an exception through the C caller."""
    import os
    import subprocess
    import sys
    from conftest import ROOT
    from test_cabi_load import _NO_MEMORY
    src, shim = tmp_path / "none.cc", tmp_path / "none.so"
    src.write_text(_NO_MEMORY)
    subprocess.check_call(["g++", "-shared", "-fPIC", "-O1", "-o", str(shim), str(src)])
    r = subprocess.run([sys.executable, "-c", _CALLS, str(shim)], cwd=ROOT, env=dict(os.environ, LD_PRELOAD=str(shim)), capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-500:]
    assert r.stdout.strip() == "%s %d" % ([_lib.ERR_NOMEM] * 7, _lib.ERR_INVALID)


@gpu
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("side,requests,N,K,top_k,group", [("head", 40, 136, 512, 1, 1), ("up", 300, 264, 128, 1, 1), ("head", 3000, 512, 256, 1, 1), ("down", 300, 136, 256, 2, 1),
                                                           ("down", 3000, 256, 128, 2, 1), ("up", 30, 264, 256, 1, 64), ("head", 60, 50, 45, 1, 1)])
def test_falling_offsets(lib, side, requests, N, K, top_k, group, int8):
    """An offset below one ahead of it counts as that one: every slot has one expert, whatever lies behind the fall."""
    S = requests * top_k
    for bad in ([0, S, 0, S, 0, S, 0], [0, 10, 5, 20, 2 ** 31 - 1, -7, S], [0, 0, S // 2, 3, S // 2 + 3, 1, S]):
        c = Experts(lib, side, requests, N, K, 6, top_k, group, 1, int8, ids=torch.arange(S).view(requests, top_k) % 6, res=side == "down")
        at = torch.tensor(bad, device="cuda")
        given = at.int()
        c.offsets = at.clamp(0, S).cummax(0).values.int()
        c.d.offsets = given.data_ptr()
        c.run().check()


@gpu
@pytest.mark.parametrize("prec", [0, 1, 2])
@pytest.mark.parametrize("act", [oracle.ACT_NONE, oracle.ACT_MISH, oracle.ACT_SELU])
@pytest.mark.parametrize("top_k", [1, 2])
def test_int8_rows_do_not_depend_on_their_number(lib, prec, act, top_k):
    """The same bits by gathers, from rows in order, and by CTA pairs, with weights and a residual."""
    made = lambda: Experts(lib, "head", 3000, 264, 512, 6, top_k, 1, prec, True, act=act, res=True, seed=5)
    whole = made().run()
    whole.check()
    for n in (1, 40, 300):
        part = made()
        part.requests = part.M = part.d.M = n
        key = torch.where(part.ids[:n] < 0, 6, part.ids[:n].long()).reshape(-1)
        part.order = torch.argsort(key, stable=True).int()
        part.offsets = torch.cat([key.new_zeros(1), torch.bincount(key, minlength=7)[:6].cumsum(0)]).int()
        part.d.order, part.d.offsets = part.order.data_ptr(), part.offsets.data_ptr()
        part.run()
        assert torch.equal(part.out[:n], whole.out[:n]) and (part.out[n:] == 55).all()


@gpu
@pytest.mark.parametrize("side", ["head", "down", "slots"])
@pytest.mark.parametrize("requests,N,experts,top_k", [(1, 1858, 6, 1), (40, 264, 6, 1), (40, 264, 6, 2), (96, 1858, 12, 1), (333, 1858, 6, 1), (2500, 256, 6, 2)])
@pytest.mark.parametrize("prec", [1, 2])
def test_float_results_are_as_exact_as_a_chain_in_fp32(lib, side, requests, N, experts, top_k, prec):
    """In the root mean square, by gathers, from rows in order, with K cut over a cluster, with choices summed.  Products of two 16-bit numbers are exact
    in fp32; a chain of 1024 rounded sums is off by about 9 2^-24 of the result's size, sums of 64 truncated at every 16 and added rounded by 2 2^-24,
    sums truncated all the way by 28 2^-24."""
    K = 1024
    ids = (torch.arange(requests)[:, None] + torch.arange(top_k) * 2) % experts
    c = Experts(lib, side, requests, N, K, experts, top_k, 1, prec, f32=True, weights=False, ids=ids, seed=9).run()
    c.check()
    want, _, written = c.want()
    chain, at = torch.zeros_like(c.out), c.offsets.tolist()
    for e in range(experts):
        choice, slot = c.order[at[e]:at[e + 1]].long(), torch.arange(at[e], at[e + 1], device="cuda")
        x, w = c.x[slot if c.from_slots else choice // top_k].float(), c.w[e * N:(e + 1) * N].float()
        y = torch.zeros(len(slot), N, device="cuda")
        for k in range(K):
            y += x[:, k, None] * w[:, k]
        chain.index_add_(0, slot if c.by_slot else choice // top_k, y + c.bias[e])
    rms = lambda v: (v.double() - want)[written].square().mean().sqrt().item()
    assert rms(c.out) <= 1.5 * rms(chain) + 2.0 ** -26


@gpu
@pytest.mark.parametrize("act", [oracle.ACT_MISH, oracle.ACT_SWISH])
@pytest.mark.parametrize("requests", [60, 900, 6000])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("worst", [NAN, INF, -INF])
def test_columns_that_share_a_reciprocal_keep_apart(lib, act, requests, int8, worst):
    c = Experts(lib, "head", requests, 264, 256, 4, 1, 1, 2, int8, act=act, weights=False, ids=torch.arange(requests)[:, None] % 4)
    clean, columns, theirs = c.bias.clone(), [5, 130, 263], torch.arange(requests, device="cuda") % 4 == 2
    c.bias[2, columns] = worst
    c.run()
    for col in columns:
        assert (c.out[theirs, col] == INF).all() if worst == INF else c.out[theirs, col].isnan().all()
    same = Experts(lib, "head", requests, 264, 256, 4, 1, 1, 2, int8, act=act, weights=False, ids=torch.arange(requests)[:, None] % 4).run()
    c.bias = clean
    for col in columns:
        c.out[theirs, col] = same.out[theirs, col]
    c.check()


@gpu
@pytest.mark.parametrize("pads", [(16, 32, 8), (0, 0, 2), (8, 0, 1), (0, 16, 0)])
@pytest.mark.parametrize("side,top_k", [("up", 2), ("down", 1), ("down", 2), ("head", 1), ("slots", 1)])
@pytest.mark.parametrize("N", [264, 1858])
@pytest.mark.parametrize("prec,int8", [(1, False), (2, False), (2, True), (0, True)])
def test_strides_of_many_rows(lib, pads, side, top_k, N, prec, int8):
    """CTA pairs: padded rows of each operand; results and residuals by whole 16 bytes, by words and by entries."""
    res = side in ("down", "head")
    pads = (2 * pads[0], *pads[1:]) if int8 else pads
    Experts(lib, side, 6000, N, 192, 5, top_k, 1, prec, int8, pads=pads, res=res, in_place=res and N == 264).run().check()


@gpu
@pytest.mark.parametrize("side", ["up", "down", "head"])
@pytest.mark.parametrize("group", [128, 192])
@pytest.mark.parametrize("requests,N", [(2, 136), (40, 520)])
@pytest.mark.parametrize("int8", [False, True])
def test_requests_of_several_whole_64_rows(lib, side, group, requests, N, int8):
    Experts(lib, side, requests, N, 256, 3, 1, group, 1, int8, res=side != "up").run().check()
    Experts(lib, side, requests, N, 192, 3, 2, group, 2, int8, res=side != "up").run().check()
