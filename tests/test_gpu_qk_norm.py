"""b200_op_qk_norm_rotate against its definition in 64 bits."""
import ctypes

import pytest

from lc0_b200 import _lib

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

DT = {0: torch.float32, 1: torch.float16, 2: torch.bfloat16}
EPS = {0: 2.0 ** -24, 1: 2.0 ** -11, 2: 2.0 ** -8}  # one rounding


class Call:
    def __init__(self, lib, rows, hq, hk, depth, prec, rotate=0, interleaved=False, norm=True, gamma=True, positions=None, n_positions=64, packed=False,
                 in_place=False, pad=0, shift=0, eps=1e-6, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed + rows + hq + depth)
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
        t = DT[prec]
        width = (hq + hk) * depth + (hk * depth if packed else 0) + pad
        flat = torch.full((shift + rows * width,), 77.0, dtype=t, device="cuda")
        both = flat[shift:].view(rows, width)
        both[:, :(hq + hk) * depth] = (rnd(rows, (hq + hk) * depth) * torch.logspace(-2, 2, rows, device="cuda")[:, None]).to(t)
        self.q, self.k = both[:, :hq * depth], both[:, hq * depth:(hq + hk) * depth]
        self.q_in, self.k_in = self.q.clone(), self.k.clone()
        if in_place:
            self.qo, self.ko = self.q, self.k
        else:
            self.qo, self.ko = (torch.full((rows, h * depth + pad), 55.0, dtype=t, device="cuda")[:, :h * depth] for h in (hq, hk))
        self.gq, self.gk = (1 + 0.3 * rnd(depth), 1 + 0.3 * rnd(depth)) if gamma else (None, None)
        angle = 20 * rnd(n_positions, max(1, rotate // 2)).double()
        self.table = torch.stack([angle.cos(), angle.sin()], dim=2).float().contiguous()
        self.at = torch.arange(rows, device="cuda") % n_positions
        self.positions = None
        if positions is not None:
            self.positions = torch.as_tensor(positions, dtype=torch.int32, device="cuda")
            self.at = self.positions.long()
        self.rows, self.hq, self.hk, self.depth, self.prec, self.rotate, self.interleaved = rows, hq, hk, depth, prec, rotate, interleaved
        self.norm, self.eps, self.n_positions, self.lib, self.in_place, self.both, self.pad = norm, eps, n_positions, lib, in_place, both, pad
        p = lambda v: None if v is None else v.data_ptr()
        self.d = _lib.QkNormDesc(q=p(self.q), k=p(self.k), ldq=width, ldk=width, q_out=p(self.qo), k_out=p(self.ko), ldq_out=self.qo.stride(0) if hq else 0,
                                 ldk_out=self.ko.stride(0) if hk else 0, rows=rows, q_heads=hq, k_heads=hk, depth=depth, precision=prec, norm=int(norm), eps=eps,
                                 gamma_q=p(self.gq), gamma_k=p(self.gk), rotate=rotate, interleaved=int(interleaved), table=p(self.table) if rotate else None,
                                 n_positions=n_positions if rotate else 0, positions=p(self.positions))

    def run(self, stream=None):
        torch.cuda.synchronize()
        _lib.check(self.lib.b200_op_qk_norm_rotate(ctypes.byref(self.d), stream))
        torch.cuda.synchronize()
        return self

    def want(self, x, heads, gamma):
        """The result, and the allowance ahead of its rounding: the sum of squares and the norm's steps are depth / 8 + 12 fp32 roundings at most
        (eight entries in a lane, five exchanges, four more), the turn two of each product's size."""
        v = x.double().reshape(self.rows, heads, self.depth)
        err = torch.zeros_like(v)
        if self.norm:
            v = v / torch.sqrt(v.square().mean(dim=2, keepdim=True) + self.eps)
            if gamma is not None:
                v = v * gamma.double()
            err = (8 + 5 + 6) * 2.0 ** -24 * v.abs()
        r = self.rotate
        if r:
            inside = ((self.at >= 0) & (self.at < self.n_positions))[:, None, None]
            turn = self.table.double()[self.at.clamp(0, self.n_positions - 1)][:, None]
            cos, sin = torch.where(inside, turn[..., 0], 1.0), torch.where(inside, turn[..., 1], 0.0)
            ia, ib = (slice(0, r, 2), slice(1, r, 2)) if self.interleaved else (slice(0, r // 2), slice(r // 2, r))
            a, b, ea, eb = v[..., ia].clone(), v[..., ib].clone(), err[..., ia].clone(), err[..., ib].clone()
            v[..., ia], v[..., ib] = a * cos - b * sin, a * sin + b * cos
            err[..., ia] = ea * cos.abs() + eb * sin.abs() + 2 * 2.0 ** -24 * ((a * cos).abs() + (b * sin).abs())
            err[..., ib] = ea * sin.abs() + eb * cos.abs() + 2 * 2.0 ** -24 * ((a * sin).abs() + (b * cos).abs())
        return v.reshape(self.rows, -1), err.reshape(self.rows, -1)

    def check(self):
        for out, x, heads, gamma in ((self.qo, self.q_in, self.hq, self.gq), (self.ko, self.k_in, self.hk, self.gk)):
            if heads == 0:
                continue
            want, err = self.want(x, heads, gamma)
            allowed = EPS[self.prec] * (want.abs() + err) + err + (2.0 ** -25 if self.prec == 1 else 1e-37)
            off = (out.double() - want).abs() / allowed
            assert off.max().item() <= 1, off.max().item()
            if not self.in_place:
                assert torch.equal(x, self.q if out is self.qo else self.k)
        assert (self.both[:, (self.hq + self.hk) * self.depth:] == 77).all()


@gpu
@pytest.mark.parametrize("prec", [0, 1, 2])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,hq,hk,depth,rotate", [(1, 1, 1, 2, 2), (1, 1, 0, 1, 0), (64, 32, 32, 32, 32), (65, 4, 2, 64, 32), (3, 5, 1, 96, 96), (200, 8, 8, 128, 64),
                                                     (130, 7, 3, 24, 8), (17, 3, 3, 30, 10), (64, 2, 1, 256, 256), (9, 1, 1, 250, 250), (1000, 24, 24, 32, 16),
                                                     (40, 16, 4, 16, 16), (33, 0, 4, 8, 8), (5000, 12, 12, 64, 64), (7, 3, 2, 200, 48)])
def test_norm_and_turn(lib, prec, interleaved, rows, hq, hk, depth, rotate):
    Call(lib, rows, hq, hk, depth, prec, rotate, interleaved).run().check()


@gpu
@pytest.mark.parametrize("prec", [0, 1, 2])
@pytest.mark.parametrize("depth,rotate,interleaved", [(32, 32, False), (32, 16, True), (64, 0, False), (20, 12, False), (20, 12, True)])
def test_packed_and_in_place(lib, prec, depth, rotate, interleaved):
    Call(lib, 192, 6, 6, depth, prec, rotate, interleaved, packed=True, in_place=True).run().check()
    Call(lib, 192, 6, 3, depth, prec, rotate, interleaved, packed=True).run().check()
    Call(lib, 50, 6, 3, depth, prec, rotate, interleaved, pad=3, shift=1, in_place=True).run().check()
    Call(lib, 50, 6, 3, depth, prec, rotate, interleaved, pad=5).run().check()


@gpu
@pytest.mark.parametrize("depth", [32, 22])
def test_parts_alone_and_positions(lib, depth):
    """No norm, no gamma, positions of their own: in any order, repeated, outside the table (not turned)."""
    Call(lib, 100, 4, 4, depth, 0, depth, norm=False).run().check()
    Call(lib, 100, 4, 4, depth, 1, depth, gamma=False).run().check()
    Call(lib, 100, 4, 4, depth, 2, 0, norm=False).run().check()
    at = torch.randint(-3, 303, (100,)).tolist()
    at[:4] = [0, 299, -1, 300]
    Call(lib, 100, 4, 2, depth, 0, depth, positions=at, n_positions=300).run().check()
    Call(lib, 100, 4, 2, depth, 1, depth - 6, positions=at, n_positions=300, interleaved=True).run().check()
    Call(lib, 4, 4, 2, depth, 0, depth, positions=[2 ** 31 - 1, 70000, -2 ** 31, 69999], n_positions=70000).run().check()


@gpu
@pytest.mark.parametrize("depth,interleaved", [(32, False), (32, True), (30, False)])
def test_zeros_and_what_is_not_finite(lib, depth, interleaved):
    """A row of zeros stays zero; NaN and infinities stay in their head, and without the norm in their pair."""
    for norm in (True, False):
        c = Call(lib, 8, 4, 4, depth, 0, 16, interleaved, norm=norm)
        c.q[0], c.q[1, depth], c.k[2, 2 * depth + 20] = 0, float("nan"), float("inf")
        c.run()
        assert not c.qo[0].any()
        bad = torch.zeros(8, 4 * depth, dtype=torch.bool, device="cuda")
        if norm:
            bad[1, depth:2 * depth] = True
        else:
            bad[1, [depth, depth + (1 if interleaved else 8)]] = True
        assert torch.equal(~c.qo.isfinite(), bad)
        bad[:] = False
        bad[2, 2 * depth + 20] = True  # the norm of an infinity: zeros beside a NaN; behind what turns
        assert torch.equal(~c.ko.isfinite(), bad)


@gpu
@pytest.mark.parametrize("depth", [8, 16, 64])
@pytest.mark.parametrize("shift", [0, 1])
def test_float_heads_by_operations_rounded_to_nearest(lib, depth, shift):
    """Entries of one size a < 2^9: the sum of squares (18 bits and 6 more), its mean and that one's root a are exact, 1 / a and a (1 / a) are
    rounded to nearest.  a (1 / a) lies within 2^-24 of 1, so the result is 1 or its neighbour below."""
    a = torch.arange(256, 512, device="cuda").float()[:, None, None]
    c = Call(lib, 256, 2, 1, depth, 0, gamma=False, eps=0.0, shift=shift)
    for v, heads in ((c.q, 2), (c.k, 1)):
        v.copy_((a * (1 - 2 * torch.randint(0, 2, (256, heads, depth), device="cuda"))).view(256, -1))
    c.run()
    for out, v in ((c.qo, c.q), (c.ko, c.k)):
        size = out * v.sign()
        assert ((size == 1) | (size == 1 - 2.0 ** -24)).all()


@gpu
def test_offsets_beyond_32_bits(lib):
    rows = 560000
    q = torch.ones(rows, 4096, dtype=torch.float16, device="cuda")
    q[-64:].normal_()
    c = Call(lib, 64, 32, 0, 128, 1, 128)
    c.q_in = q[-64:].clone()
    out = torch.empty_like(q)
    c.d.q, c.d.q_out, c.d.ldq, c.d.ldq_out, c.d.rows = q.data_ptr(), out.data_ptr(), 4096, 4096, rows
    c.run()
    c.q, c.qo = q[-64:], out[-64:]
    c.check()


@gpu
def test_captured_and_on_a_stream(lib):
    c = Call(lib, 640, 12, 12, 32, 1, 32)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    _lib.check(lib.b200_op_qk_norm_rotate(ctypes.byref(c.d), st.cuda_stream))
    st.synchronize()
    c.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        _lib.check(lib.b200_op_qk_norm_rotate(ctypes.byref(c.d), torch.cuda.current_stream().cuda_stream))
    c.q.mul_(-2)
    c.q_in.copy_(c.q)
    graph.replay()
    torch.cuda.synchronize()
    c.check()


def test_refusals(lib):
    def call(**kw):
        d = _lib.QkNormDesc(q=256, k=256, q_out=512, k_out=512, rows=4, q_heads=2, k_heads=2, depth=32, precision=1, norm=1, eps=1e-6, rotate=32, table=256,
                            n_positions=64)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.b200_op_qk_norm_rotate(ctypes.byref(d), None)

    assert lib.b200_op_qk_norm_rotate(None, None) == _lib.ERR_INVALID
    assert call(rows=0) == _lib.OK and call(q_heads=0, k_heads=0) == _lib.OK
    for kw in (dict(rows=-1), dict(q_heads=-1), dict(k_heads=-1), dict(depth=0), dict(depth=257), dict(precision=3), dict(eps=-1.0), dict(eps=float("nan")),
               dict(rotate=33), dict(rotate=34), dict(rotate=-2), dict(n_positions=0), dict(table=None), dict(q=None), dict(k=None), dict(q_out=None),
               dict(k_out=None), dict(ldq=63), dict(ldk=1), dict(ldq_out=63), dict(ldk_out=1), dict(q=257), dict(k_out=513), dict(gamma_q=258), dict(gamma_k=257),
               dict(table=260), dict(positions=257), dict(q_out=256, ldq_out=128), dict(k_out=256, ldk=96), dict(rows=2 ** 30)):
        assert call(**kw) == _lib.ERR_INVALID, kw
        assert b"b200_op_qk_norm_rotate" in lib.b200_last_error()
