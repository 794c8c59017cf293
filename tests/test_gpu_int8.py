"""b200_op_quantize_rows and b200_op_gemm_int8 against their definitions in 64 bits."""
import ctypes

import pytest

from lc0_b200 import _lib
from oracle import oracle

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

DT = {0: torch.float32, 1: torch.float16, 2: torch.bfloat16}
EPS = {0: 2.0 ** -24, 1: 2.0 ** -11, 2: 2.0 ** -8}  # one rounding
SLOPE = {oracle.ACT_NONE: 1.0, oracle.ACT_RELU: 1.0, oracle.ACT_MISH: 1.1, oracle.ACT_SWISH: 1.1, oracle.ACT_TANH: 1.0,
         oracle.ACT_SIGMOID: 0.25, oracle.ACT_SELU: 1.76}
INF, NAN = float("inf"), float("nan")


def activate(v, act):
    f = torch.nn.functional
    return {oracle.ACT_NONE: lambda x: x, oracle.ACT_RELU: torch.relu, oracle.ACT_MISH: f.mish, oracle.ACT_SWISH: f.silu,
            oracle.ACT_RELU_2: lambda x: torch.relu(x) ** 2, oracle.ACT_TANH: torch.tanh, oracle.ACT_SIGMOID: torch.sigmoid,
            oracle.ACT_SELU: f.selu}[act](v)


def activated(y, err, act, fast):
    """act(y) and what an error of `err` in y and the arithmetic of the activation can make of it (16-bit results use __expf and __fdividef,
    others expf: a few steps of the argument's size)."""
    want = activate(y, act)
    err = 2 * y.abs() * err + err * err if act == oracle.ACT_RELU_2 else SLOPE[act] * err
    if act == oracle.ACT_RELU_2:
        err = err + 2.0 ** -24 * want
    elif act not in (oracle.ACT_NONE, oracle.ACT_RELU):
        err = err + (2.0 ** -17 if fast else 2.0 ** -20) * (want.abs() + 1e-2 * y.abs())
        if act == oracle.ACT_SELU:
            # 1.76 (exp(y) - 1) below zero: exp is off by two steps (__expf: by 2 + 1.2 |y|), which are 2^-24 below one, and the difference with
            # one is exact from 1/2 up and rounded by one more step of that size at most below
            err = err + torch.where(y < 0, 1.76 * 2.0 ** -24 * ((4 if fast else 3) + (1.2 * y.abs().clamp(max=20) if fast else 0)), 0.0)
    return want, err


def rows(r, c, pad, value, fill, shift=0):
    """`value` as rows with a gap behind each, behind an odd start."""
    flat = torch.full((shift + r * (c + pad),), fill, dtype=value.dtype, device="cuda")
    t = flat[shift:].view(r, c + pad)[:, :c]
    t.copy_(value)
    return t


def quantize(lib, x, pad=0, shift=0, stream=None):
    m, k = x.shape
    q = rows(m, k, pad, torch.zeros(m, k, dtype=torch.int8, device="cuda"), 77, shift)
    s = torch.full((m,), 7.0, device="cuda")
    torch.cuda.synchronize()
    _lib.check(lib.b200_op_quantize_rows(x.data_ptr(), x.stride(0), m, k, {v: n for n, v in DT.items()}[x.dtype], q.data_ptr(), q.stride(0), s.data_ptr(), stream))
    torch.cuda.synchronize()
    if pad and m > 1:
        assert (torch.as_strided(q, (m - 1, pad), (k + pad, 1), q.storage_offset() + k) == 77).all()
    return q, s


def quantized(x):
    """The definition: the scale is a number of 32 bits, the quotient that of 64 (which a tie of two 24-bit numbers cannot miss)."""
    s = x.float().abs().amax(dim=1) * torch.tensor(1 / 127, device=x.device)
    bad = ~x.float().isfinite().all(dim=1)
    ok = (s > 0) & ~bad
    q = torch.round(x.double() / torch.where(ok, s, 1.0).double()[:, None]).clamp(-127, 127)
    return torch.where(ok[:, None], q, 0.0).to(torch.int8), torch.where(bad, NAN, s)


@gpu
@pytest.mark.parametrize("prec", [0, 1, 2])
@pytest.mark.parametrize("m,k,pad,shift", [(1, 1, 0, 0), (3, 7, 1, 1), (64, 8, 0, 0), (5, 64, 8, 0), (33, 256, 0, 0), (64, 1024, 16, 0), (7, 1000, 0, 0), (9, 1536, 0, 8),
                                           (130, 2048, 8, 0), (6, 2056, 0, 0), (3, 5000, 0, 0), (2, 40000, 0, 0), (1000, 72, 0, 0), (11, 513, 3, 5)])
def test_quantize_rows(lib, prec, m, k, pad, shift):
    g = torch.Generator(device="cuda").manual_seed(m + 3 * k)
    v = torch.randn(m, k, device="cuda", generator=g) * torch.logspace(-3, 3, m, device="cuda")[:, None].clamp(max=6e3)
    x = rows(m, k, pad, v.to(DT[prec]), NAN, shift)
    q, s = quantize(lib, x, pad, shift)
    want_q, want_s = quantized(x)
    assert torch.equal(s, want_s)
    assert torch.equal(q.contiguous(), want_q)


@gpu
@pytest.mark.parametrize("prec", [0, 1, 2])
@pytest.mark.parametrize("k", [64, 61, 4096])
def test_quantize_rows_at_the_ends(lib, prec, k):
    """Ties, the smallest and largest numbers of the type, zeros, infinities and NaN, each in a row of its own."""
    t = DT[prec]
    info = torch.finfo(t)
    x = torch.zeros(12, k, dtype=t, device="cuda")
    ramp = torch.arange(k, device="cuda") % 250
    x[1] = (ramp - 124.5).to(t)
    x[1, 0] = 127  # scale 1 but for its last bit: quotients beside ties
    x[2] = (ramp - 125).to(t) * 0.5
    x[2, 1] = -127
    x[3] = info.max
    x[4, ::3] = info.tiny * info.eps  # the smallest subnormal number
    x[5] = info.tiny * (1 + ramp.to(t) / 256)
    x[6] = 1.0
    x[6, k - 1] = INF
    x[7, 0] = NAN
    x[8, k // 2] = -INF
    x[9] = -info.max
    x[9, 5] = info.tiny
    x[10] = 3.0
    x[11] = torch.linspace(-1, 1, k, device="cuda").to(t) * info.max
    q, s = quantize(lib, x)
    want_q, want_s = quantized(x)
    assert torch.equal(s.nan_to_num(-1.0), want_s.nan_to_num(-1.0))
    assert torch.equal(q, want_q)
    assert s[6:9].isnan().all() and not q[6:9].any() and s[0] == 0


@gpu
@pytest.mark.parametrize("k", [768, 765])
def test_quotients_a_step_from_a_tie(lib, k):
    """fp32 rows whose scales lie at both ends of a binade and anywhere in it, of many sizes, with entries at (r + 1/2) s rounded and one step to
    either side: what the remainder alone decides."""
    ends = [1.0, 1 + 2.0 ** -23, 1 + 3 * 2.0 ** -23, 1.5, 2 - 2.0 ** -22, 2 - 2.0 ** -23]
    some = (1 + torch.rand(58, dtype=torch.float64, generator=torch.Generator().manual_seed(k))).tolist()
    most = torch.tensor([127 * s * 2.0 ** e for s in ends + some for e in (-110, -97, -20, 0, 3, 60, 119)], dtype=torch.float64, device="cuda").float()
    scale = most * torch.tensor(1 / 127, device="cuda")
    tie = ((torch.arange(-127, 127, device="cuda") + 0.5).double() * scale.double()[:, None]).float()
    inf = torch.full_like(tie, INF)
    x = torch.cat([tie, torch.nextafter(tie, inf), torch.nextafter(tie, -inf)], dim=1)
    x = torch.cat([x, torch.zeros(len(most), 6, device="cuda")], dim=1)[:, :k].contiguous()
    x[:, k - 1] = most
    assert (x.abs().amax(dim=1) == most).all()
    q, s = quantize(lib, x)
    want_q, want_s = quantized(x)
    assert torch.equal(s, want_s) and torch.equal(q, want_q)


class Product:
    def __init__(self, lib, M, N, K, prec, act=oracle.ACT_NONE, bias=True, res=True, alpha=1.0, pads=(0, 0, 0), shift=0, seed=0, in_place=False):
        g = torch.Generator(device="cuda").manual_seed(seed + M + 3 * N + 7 * K)
        whole = lambda *s: torch.randint(-127, 128, s, device="cuda", generator=g).to(torch.int8)
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
        self.x, self.w = rows(M, K, pads[0], whole(M, K), 99, shift), rows(N, K, pads[1], whole(N, K), 99, shift)
        self.sx, self.sw = (0.5 + torch.rand(M, device="cuda", generator=g)) / 73, (0.5 + torch.rand(N, device="cuda", generator=g)) / 73 * K ** -0.5
        self.bias = rnd(N) if bias else None
        self.out = rows(M, N, pads[2], torch.zeros(M, N, dtype=DT[prec], device="cuda"), 77.0, shift)
        self.res = None
        if res:
            self.res = rows(M, N, pads[2], rnd(M, N).to(DT[prec]), NAN, shift)
            if in_place:
                self.out.copy_(self.res)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.M, self.N, self.K, self.prec, self.act, self.alpha, self.lib = M, N, K, prec, act, alpha, lib
        p = lambda v: None if v is None else v.data_ptr()
        self.d = _lib.GemmInt8Desc(X=p(self.x), x_scales=p(self.sx), W=p(self.w), w_scales=p(self.sw), bias=p(self.bias), C=p(self.out), M=M, N=N, K=K,
                                   ldx=self.x.stride(0), ldw=self.w.stride(0), ldc=self.out.stride(0), activation=act, precision=prec, alpha=alpha,
                                   res=p(self.out if in_place else self.res), ldres=self.out.stride(0), status=p(self.status))

    def run(self, stream=None):
        torch.cuda.synchronize()
        _lib.check(self.lib.b200_op_gemm_int8(ctypes.byref(self.d), stream))
        torch.cuda.synchronize()
        assert self.status.item() == 0
        return self

    def check(self):
        """Whole sums are exact; their conversion, the scales' product, that with the sum, and the bias are one fp32 rounding each."""
        scaled = (self.x.double() @ self.w.double().T) * (self.sx.double()[:, None] * self.sw.double())
        y, mag = scaled, scaled.abs()
        if self.bias is not None:
            y, mag = y + self.bias.double(), mag + self.bias.double().abs()
        want, err = activated(y, 4 * 2.0 ** -24 * mag, self.act, self.prec != 0)
        want, err = want * self.alpha, (err + 2.0 ** -24 * want.abs()) * abs(self.alpha)
        if self.res is not None:
            want = want + self.res.double()
            err = err + 2.0 ** -24 * (want.abs() + err)
        allowed = EPS[self.prec] * (want.abs() + err) + err + (2.0 ** -25 if self.prec == 1 else 1e-37)
        off = (self.out.double() - want).abs() / allowed
        assert off.max().item() <= 1, off.max().item()  # NaN fails
        if self.out.stride(0) > self.N and self.M > 1:
            gap = torch.as_strided(self.out, (self.M - 1, self.out.stride(0) - self.N), (self.out.stride(0), 1), self.out.storage_offset() + self.N)
            assert (gap == 77).all()


SHAPES = [(1, 1, 1), (1, 8, 16), (2, 130, 45), (31, 64, 64), (64, 1024, 1024), (65, 96, 64), (37, 1858, 2048), (128, 128, 128), (129, 257, 144), (200, 264, 136),
          (256, 256, 512), (300, 1000, 624), (513, 520, 320), (1000, 32, 256), (1536, 1536, 1024), (4096, 768, 256), (20000, 512, 128), (16384, 1024, 1536),
          (333, 1858, 1024), (70000, 16, 32), (300, 1, 64), (60, 3, 128), (5000, 5, 64), (2000, 129, 64), (6000, 385, 256)]


@gpu
@pytest.mark.parametrize("prec", [0, 1, 2])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(lib, prec, M, N, K):
    Product(lib, M, N, K, prec, act=[oracle.ACT_NONE, oracle.ACT_MISH, oracle.ACT_RELU_2][(M + prec) % 3], res=(M + N + prec) % 2 == 0).run().check()


@gpu
@pytest.mark.parametrize("act", sorted(SLOPE) + [oracle.ACT_RELU_2])
@pytest.mark.parametrize("prec", [0, 1, 2])
@pytest.mark.parametrize("M", [37, 700])
def test_activations(lib, act, prec, M):
    Product(lib, M, 264, 256, prec, act=act, alpha=0.75, seed=act).run().check()


@gpu
@pytest.mark.parametrize("pads,shift", [((16, 32, 8), 0), ((5, 0, 0), 0), ((0, 3, 1), 0), ((0, 0, 3), 1), ((16, 16, 8), 16)])
@pytest.mark.parametrize("M,N,K", [(65, 200, 256), (700, 384, 512), (33, 50, 1040)])
@pytest.mark.parametrize("prec", [0, 1])
def test_strides(lib, pads, shift, M, N, K, prec):
    Product(lib, M, N, K, prec, pads=pads, shift=shift).run().check()


@gpu
@pytest.mark.parametrize("M,N,K,prec", [(64, 1024, 512, 1), (3000, 1024, 512, 2), (37, 333, 100, 0)])
def test_residual_in_place(lib, M, N, K, prec):
    Product(lib, M, N, K, prec, in_place=True, alpha=-0.5).run().check()
    Product(lib, M, N, K, prec, bias=False, res=False).run().check()


@gpu
@pytest.mark.parametrize("M,N,K", [(40, 64, 131071), (300, 48, 131056), (40, 64, 131056)])
def test_longest_sums_do_not_overflow(lib, M, N, K):
    p = Product(lib, M, N, K, 0, bias=False, res=False)
    p.x.fill_(127)
    p.w.fill_(-127)
    p.w[::2] = 127
    p.run().check()


@gpu
def test_rows_do_not_depend_on_their_number(lib):
    whole = Product(lib, 5000, 520, 1024, 1, act=oracle.ACT_MISH, seed=1).run()
    for m in (1, 33, 64, 200, 1500):
        part = Product(lib, 5000, 520, 1024, 1, act=oracle.ACT_MISH, seed=1)
        part.d.M = m
        part.run()
        assert torch.equal(part.out[:m], whole.out[:m]) and not part.out[m:].any()  # rows behind the last are left as they were


@gpu
@pytest.mark.parametrize("act", [oracle.ACT_NONE, oracle.ACT_MISH, oracle.ACT_SWISH, oracle.ACT_RELU_2, oracle.ACT_SELU])
@pytest.mark.parametrize("prec", [0, 1, 2])
def test_rows_do_not_depend_on_their_number_whatever_follows(lib, act, prec):
    """The same bits from each kernel with alpha, bias and residual: a cluster per tile, a tile per CTA, CTA pairs with narrow and with wide tiles."""
    made = lambda: Product(lib, 6000, 520, 1024, prec, act=act, alpha=-0.7, seed=2)
    whole = made().run()
    whole.check()
    for m in (1, 64, 500, 3000):
        part = made()
        part.d.M = m
        part.run()
        assert torch.equal(part.out[:m], whole.out[:m]) and not part.out[m:].any()


@gpu
@pytest.mark.parametrize("pads", [(16, 32, 8), (0, 0, 2), (48, 0, 1), (0, 16, 0)])
@pytest.mark.parametrize("M,N,K", [(3000, 520, 256), (6000, 520, 336), (3000, 1858, 144), (6000, 1857, 128)])
@pytest.mark.parametrize("prec", [0, 1, 2])
def test_strides_of_many_rows(lib, pads, M, N, K, prec):
    """CTA pairs: padded rows of each operand; results and residuals by whole 16 bytes, by words and by entries, in narrow and in wide tiles."""
    act = oracle.ACT_MISH if pads[2] == 2 else oracle.ACT_NONE
    Product(lib, M, N, K, prec, pads=pads, act=act).run().check()
    Product(lib, M, N, K, prec, pads=pads, in_place=True).run().check()
    Product(lib, M, N, K, prec, pads=pads, res=False, alpha=0.5).run().check()


@gpu
@pytest.mark.parametrize("act", [oracle.ACT_MISH, oracle.ACT_SWISH])
@pytest.mark.parametrize("M", [64, 500, 3000])
@pytest.mark.parametrize("prec", [1, 2])
@pytest.mark.parametrize("worst", [NAN, INF, -INF])
def test_columns_that_share_a_reciprocal_keep_apart(lib, act, M, prec, worst):
    """Four columns of a row share the activation's reciprocal; one that is not finite reaches none of the others."""
    p = Product(lib, M, 300, 256, prec, act=act, res=False)
    clean = p.bias.clone()
    p.bias[7], p.bias[12], p.bias[298] = worst, worst, worst
    p.run()
    bad = [7, 12, 298]
    if worst != INF:
        assert p.out[:, bad].isnan().all()
    else:
        assert (p.out[:, bad] == (65504 if prec == 1 else INF)).all()
    p.out[:, bad] = Product(lib, M, 300, 256, prec, act=act, res=False).run().out[:, bad]
    p.bias = clean
    p.check()


@gpu
def test_offsets_beyond_32_bits(lib):
    """Rows whose entries, and whose bytes, lie more than 2^32 behind the first."""
    M, N, K = 600000, 4096, 32
    p = Product(lib, 64, N, K, 1, res=False)
    x, out = torch.zeros(M, K, dtype=torch.int8, device="cuda"), torch.empty(M, N, dtype=torch.float16, device="cuda")
    sx = torch.ones(M, device="cuda")
    x[-64:], sx[-64:] = p.x, p.sx
    p.d.X, p.d.x_scales, p.d.C, p.d.M = x.data_ptr(), sx.data_ptr(), out.data_ptr(), M
    p.run()
    p.out = out[-64:]
    p.check()
    del out
    wide = torch.empty(33000, 131072 // 2, dtype=torch.float16, device="cuda")
    wide[-1].normal_()
    wide[:-1] = 1
    q, s = quantize(lib, wide)
    assert torch.equal(q[-1:], quantized(wide[-1:])[0]) and torch.equal(s[-1:], quantized(wide[-1:])[1]) and (q[-2] == 127).all()


@gpu
def test_scales_that_are_not_numbers_stay_in_their_row_and_column(lib):
    for M in (64, 900):
        p = Product(lib, M, 300, 256, 1, res=False)
        p.sx[5], p.sw[7] = NAN, NAN
        p.run()
        bad = torch.zeros(M, 300, dtype=torch.bool, device="cuda")
        bad[5], bad[:, 7] = True, True
        assert torch.equal(p.out.isnan(), bad)


@gpu
def test_streams_and_graphs(lib):
    """A layer in 8 bits captured once and replayed with other activations; two such graphs on two streams; and a side stream."""
    M, N, K = 640, 512, 768
    p = [Product(lib, M, N, K, 2, seed=i) for i in (1, 2)]
    xs = [torch.randn(M, K, device="cuda").to(torch.bfloat16) for _ in p]
    streams, graphs = [torch.cuda.Stream() for _ in p], []
    torch.cuda.synchronize()

    def layer(i):
        st = torch.cuda.current_stream().cuda_stream
        _lib.check(lib.b200_op_quantize_rows(xs[i].data_ptr(), 0, M, K, 2, p[i].x.data_ptr(), p[i].x.stride(0), p[i].sx.data_ptr(), st))
        _lib.check(lib.b200_op_gemm_int8(ctypes.byref(p[i].d), st))

    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            layer(i)
        st.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            layer(i)
        graphs.append(graph)
    for turn in range(3):
        for x in xs:
            x.normal_()
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            q, s = quantized(xs[i])
            assert torch.equal(p[i].x, q) and torch.equal(p[i].sx, s)
            p[i].check()


def test_quantize_refusals(lib):
    call = lib.b200_op_quantize_rows
    good = [256, 0, 4, 64, 1, 256, 0, 256, None]
    assert call(None, 0, 0, 64, 1, None, 0, None, None) == _lib.OK  # no rows: nothing to do
    for at, v in ((0, None), (0, 257), (1, 63), (2, -1), (3, 0), (4, 3), (4, -1), (5, None), (6, 10), (7, None), (7, 258)):
        assert call(*[v if i == at else a for i, a in enumerate(good)]) == _lib.ERR_INVALID, (at, v)
        assert b"b200_op_quantize_rows" in lib.b200_last_error()


def test_product_refusals(lib):
    def call(**kw):
        d = _lib.GemmInt8Desc(X=256, x_scales=256, W=256, w_scales=256, C=256, M=4, N=8, K=64, activation=3, precision=1, alpha=1.0)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.b200_op_gemm_int8(ctypes.byref(d), None)

    assert lib.b200_op_gemm_int8(None, None) == _lib.ERR_INVALID
    assert call(M=0) == _lib.OK
    for kw in (dict(X=None), dict(W=None), dict(C=None), dict(x_scales=None), dict(w_scales=None), dict(M=-1), dict(N=0), dict(K=0), dict(K=131072),
               dict(precision=3), dict(precision=-1), dict(activation=0), dict(activation=9), dict(ldx=63), dict(ldw=1), dict(ldc=7), dict(res=256, ldres=7),
               dict(C=257), dict(x_scales=258), dict(w_scales=258), dict(bias=258), dict(res=257), dict(status=258), dict(res=256, ldres=16)):
        assert call(**kw) == _lib.ERR_INVALID, kw
        assert b"b200_op_gemm_int8" in lib.b200_last_error()
