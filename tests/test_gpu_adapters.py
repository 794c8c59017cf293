"""b200_op_gemm_adapters against products in 64 bits."""
import ctypes

import numpy as np
import pytest

from lc0_b200 import _lib
from oracle import oracle

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

DT = {0: torch.float32, 1: torch.float16, 2: torch.bfloat16}
EPS = {0: 2.0 ** -24, 1: 2.0 ** -11, 2: 2.0 ** -8}     # one rounding
PIECES = {0: 0.0, 1: 2.0 ** -22, 2: 2.0 ** -16}        # X A^T as two values of the type: the second one's rounding
TINY = {0: 0.0, 1: 2.0 ** -25, 2: 0.0}                 # ... and where fp16's smallest numbers end
SLOPE = {oracle.ACT_NONE: 1.0, oracle.ACT_RELU: 1.0, oracle.ACT_MISH: 1.1, oracle.ACT_SWISH: 1.1, oracle.ACT_TANH: 1.0,
         oracle.ACT_SIGMOID: 0.25, oracle.ACT_SELU: 1.76}


def activate(v, act):
    f = torch.nn.functional
    return {oracle.ACT_NONE: lambda x: x, oracle.ACT_RELU: torch.relu, oracle.ACT_MISH: f.mish, oracle.ACT_SWISH: f.silu,
            oracle.ACT_RELU_2: lambda x: torch.relu(x) ** 2, oracle.ACT_TANH: torch.tanh, oracle.ACT_SIGMOID: torch.sigmoid,
            oracle.ACT_SELU: f.selu}[act](v)


class Call:
    """One call's tensors and description."""

    def __init__(self, lib, M, N, K, rank, group, adapters, prec, act=oracle.ACT_NONE, out_f32=0, bias=True, scales=True, pads=(0, 0, 0),
                 shift=0, seed=0, ids=None):
        g = torch.Generator(device="cuda").manual_seed(seed + M + 3 * N + 7 * K + rank)
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)

        def rows(r, c, pad, value, fill):  # rows with a gap behind each and an odd start
            flat = torch.full((shift + r * (c + pad),), fill, dtype=value.dtype, device="cuda")
            t = flat[shift:].view(r, c + pad)[:, :c]
            t.copy_(value)
            return t

        t = DT[prec]
        self.x = rows(M, K, pads[0], rnd(M, K).to(t), float("nan"))
        self.w = rows(N, K, pads[1], (rnd(N, K) * K ** -0.5).to(t), float("nan"))
        self.out = rows(M, N, pads[2], torch.zeros(M, N, dtype=torch.float32 if out_f32 else t, device="cuda"), 77.0)
        self.a, self.b = (rnd(adapters, rank, K) * K ** -0.5).to(t), (rnd(adapters, N, rank) * rank ** -0.5).to(t)
        self.bias = rnd(N) if bias else None
        self.scales = torch.rand(adapters, device="cuda", generator=g) + 0.5 if scales else None
        requests = (M + group - 1) // group
        if ids is None:
            ids = torch.randint(-1, adapters, (requests,), device="cuda", generator=g)
        self.ids = torch.as_tensor(ids, dtype=torch.int32, device="cuda").contiguous()
        assert self.ids.numel() == requests
        self.M, self.N, self.K, self.rank, self.group, self.adapters = M, N, K, rank, group, adapters
        self.prec, self.act, self.out_f32, self.lib = prec, act, out_f32, lib
        p = lambda v: None if v is None else v.data_ptr()
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.d = _lib.AdaptersDesc(X=p(self.x), W=p(self.w), bias=p(self.bias), C=p(self.out), M=M, N=N, K=K, ldx=self.x.stride(0),
                                   ldw=self.w.stride(0), ldc=self.out.stride(0), activation=act, precision=prec, out_f32=out_f32,
                                   A=p(self.a), B=p(self.b), scales=p(self.scales), n_adapters=adapters, rank=rank, ids=p(self.ids),
                                   group=group, status=p(self.status))
        need = ctypes.c_size_t()
        _lib.check(lib.b200_op_gemm_adapters_workspace(ctypes.byref(self.d), ctypes.byref(need)))
        self.ws = torch.full((need.value + 64,), 255, dtype=torch.uint8, device="cuda")  # NaN in every type
        self.d.workspace, self.d.workspace_bytes = self.ws.data_ptr(), need.value

    def run(self, stream=None):
        torch.cuda.synchronize()
        _lib.check(self.lib.b200_op_gemm_adapters(ctypes.byref(self.d), stream))
        torch.cuda.synchronize()
        assert self.status.item() == 0 and (self.ws[-64:] == 255).all()
        return self.out

    def want(self):
        """Sums in 64 bits, and the allowance: half a step of the output's type; sums of K and of rank products in fp32 (chains of
        K / 8, in pieces, of truncated additions), in two of which H's error is seen through B."""
        ids = self.ids.long().repeat_interleave(self.group)[:self.M]
        x, w = self.x.double(), self.w.double()
        y, mag = x @ w.T, x.abs() @ w.abs().T
        delta, dmag, tiny = torch.zeros_like(y), torch.zeros_like(y), torch.zeros_like(y)
        for j in range(self.adapters):
            r = (ids == j).nonzero()[:, 0]
            s = 1.0 if self.scales is None else self.scales[j].double()
            a, b = self.a[j].double(), self.b[j].double()
            delta[r] = s * (x[r] @ a.T @ b.T)
            dmag[r] = s * (x[r].abs() @ a.abs().T @ b.abs().T)
            tiny[r] = b.abs().sum(1)
        y, mag = y + delta, mag + delta.abs()
        if self.bias is not None:
            y, mag = y + self.bias.double(), mag + self.bias.double().abs()
        err = (self.K / 8 + 24) * 2.0 ** -24 * (mag + 2 * dmag) + PIECES[self.prec] * dmag + TINY[self.prec] * tiny
        want = activate(y, self.act)
        if self.act == oracle.ACT_RELU_2:
            err = 2 * y.abs() * err + err * err
        else:
            err = SLOPE[self.act] * err
        # activations: __expf and __fdividef (16-bit results) or expf, a few steps of the argument's size
        fast = self.prec and not self.out_f32
        err = err + (0.0 if self.act in (oracle.ACT_NONE, oracle.ACT_RELU, oracle.ACT_RELU_2) else
                     ((2.0 ** -17 if fast else 2.0 ** -20) * (want.abs() + 1e-2 * y.abs())))
        half = EPS[0] if self.out_f32 else EPS[self.prec]
        return want, half * (want.abs() + err) + err + (2.0 ** -25 if self.prec == 1 and not self.out_f32 else 1e-37)

    def check(self):
        want, allowed = self.want()
        off = (self.out.double() - want).abs() / allowed
        assert off.max().item() <= 1, off.max().item()  # NaN fails
        if self.out.stride(0) > self.N:  # what lies between the rows is left as it was
            gap = torch.as_strided(self.out, (self.M - 1, self.out.stride(0) - self.N), (self.out.stride(0), 1), self.out.storage_offset() + self.N)
            assert (gap == 77).all()


@gpu
@pytest.mark.parametrize("prec", [0, 1, 2])
@pytest.mark.parametrize("M,N,K,rank,group,adapters", [
    (1, 1, 1, 1, 1, 1), (1, 8, 8, 1, 1, 3), (3, 130, 45, 5, 1, 4), (63, 200, 72, 8, 1, 7), (64, 256, 512, 16, 64, 2), (65, 96, 64, 16, 64, 2),
    (128, 1024, 1024, 16, 64, 5), (200, 264, 136, 24, 64, 3), (1000, 256, 256, 8, 1, 50), (1024, 128, 2048, 8, 1, 16),
    (1536, 1536, 1024, 16, 64, 9), (4096, 1024, 1024, 32, 64, 20), (5000, 520, 320, 40, 64, 30), (4160, 768, 256, 64, 128, 4),
    (8192, 512, 256, 13, 192, 6), (2048, 512, 512, 128, 64, 8), (8192, 1024, 512, 128, 64, 8), (2048, 1536, 256, 96, 256, 3), (600, 300, 200, 16, 7, 11),
    (12800, 1096, 576, 48, 64, 100), (2048, 1858, 512, 16, 32, 12), (19008, 512, 256, 16, 64, 64), (6400, 320, 128, 16, 6400, 1)])
def test_shapes(lib, prec, M, N, K, rank, group, adapters):
    if prec == 0 and M * N * K > 1 << 31:
        M = group * 12
    c = Call(lib, M, N, K, rank, group, adapters, prec)
    c.run()
    c.check()


@gpu
@pytest.mark.parametrize("act", sorted(SLOPE) + [oracle.ACT_RELU_2])
@pytest.mark.parametrize("prec,out_f32", [(0, 0), (1, 0), (2, 0), (1, 1), (2, 1)])
@pytest.mark.parametrize("M,N,group", [(37, 120, 1), (256, 512, 64), (8192, 768, 64)])
def test_activations_and_fp32_results(lib, act, prec, out_f32, M, N, group):
    c = Call(lib, M, N, 256, 16, group, 9, prec, act=act, out_f32=out_f32)
    c.run()
    c.check()


@gpu
@pytest.mark.parametrize("prec", [1, 2])
@pytest.mark.parametrize("M,N,K,rank,group", [(37, 1858, 2048, 16, 1), (2000, 1858, 2048, 16, 1), (2000, 1858, 1024, 16, 1), (4000, 256, 2048, 13, 1),
                                              (1000, 1000, 512, 32, 1), (2048, 1024, 2048, 16, 64)])
def test_fp32_results_do_not_show_long_chains(lib, prec, M, N, K, rank, group):
    """A chain of n truncated additions, each at most one step (2^-23) of a sum that grows like the root of its place, is off by at
    most n 2/3 of a step of its end: chains of 256 are n = 16.  Seven joins of pieces add half a step each.  Root mean square,
    relative, of the rows that are the shared product alone (an adapter or a bias beside it would make less of it):
    (16 * 2/3 * 2 + 7) 2^-24.  One chain of 2048 measures 2.1e-6 (bf16) and 2.4e-6 (fp16)."""
    c = Call(lib, M, N, K, rank, group, 20, prec, out_f32=1, bias=False, ids=torch.arange((M + group - 1) // group) % 3 - 1)
    c.run()
    c.check()
    alone = (c.ids < 0).repeat_interleave(group)[:M]
    want = c.want()[0][alone]
    off = ((c.out[alone].double() - want).norm() / want.norm()).item()
    assert off <= (16 * 2 / 3 * 2 + 7) * 2.0 ** -24, off



def rounded(K, rank=0):
    """Relative error, root mean square, of sums whose every 64 terms are four truncated additions and whose further ones are rounded.  A
    truncation takes half a step of 2^-23 on average, 0.72 of that in relation to the sum, which grows like the root of its
    place: 0.36 (0.5 + 0.71 + 0.87 + 1) = 1.1 steps, always towards zero, so that all chains together are off by as much.  A rounding is off
    by 1 / sqrt(12) of a step, 0.43 of 2^-24 in relation to the sum; K / 64 of them, of sums that grow, and those over the ranks.  A tenth for chance."""
    return 1.1 * (2.2 ** 2 + 0.43 ** 2 * (K / 128 + rank / 2)) ** 0.5 * 2.0 ** -24


@gpu
@pytest.mark.parametrize("prec", [1, 2])
@pytest.mark.parametrize("M,N,K,group", [(37, 1858, 256, 1), (4000, 1858, 256, 1), (4000, 520, 512, 1), (1000, 1000, 1000, 1), (37, 1858, 2048, 1), (500, 1858, 4096, 1),
                                         (4000, 256, 2560, 1), (4000, 1858, 8192, 1), (2048, 1024, 256, 64), (8192, 512, 1024, 64)])
def test_fp32_results_are_as_exact_as_a_plain_product(lib, prec, M, N, K, group):
    """Of the rows without an adapter: within the error derived above or that of a product in fp32 of the same numbers (of fp16 the
    products themselves have 22 bits, and any sum of them rounds more often)."""
    c = Call(lib, M, N, K, 16, group, 20, prec, out_f32=1, bias=False, ids=torch.arange((M + group - 1) // group) % 3 - 1)
    c.run()
    c.check()
    alone = (c.ids < 0).repeat_interleave(group)[:M]
    want = c.want()[0][alone]
    plain = c.x[alone].float() @ c.w.float().T
    rms = lambda v: ((v.double() - want).norm() / want.norm()).item()
    assert rms(c.out[alone]) <= max(rounded(K), 1.05 * rms(plain)), (rms(c.out[alone]), rms(plain))


@gpu
@pytest.mark.parametrize("prec", [1, 2])
@pytest.mark.parametrize("M,N,K,rank,group", [(2048, 256, 256, 16, 64), (2048, 256, 2048, 16, 64), (4096, 264, 2048, 128, 64), (4160, 256, 8192, 40, 192),
                                              (50, 256, 2048, 16, 1)])
def test_fp32_results_of_adapters_alone(lib, prec, M, N, K, rank, group):
    """A shared product of zeros: what is left shows how X A^T was summed."""
    c = Call(lib, M, N, K, rank, group, 20, prec, out_f32=1, bias=False, ids=torch.arange((M + group - 1) // group) % 20)
    c.w.zero_()
    c.run()
    want = c.want()[0]
    x, ids = c.x.float(), c.ids.long().repeat_interleave(group)[:M]
    plain = torch.cat([c.scales[j] * (x[i:i + 1] @ c.a[j].float().T @ c.b[j].float().T) for i, j in enumerate(ids.tolist()[:200])])
    off = ((c.out.double() - want).norm() / want.norm()).item()
    of_plain = ((plain.double() - want[:200]).norm() / want[:200].norm()).item()
    assert off <= max(rounded(K, rank), 1.05 * of_plain), (off, of_plain)


@gpu
@pytest.mark.parametrize("prec", [1, 2])
@pytest.mark.parametrize("K", [256, 2048])
def test_fp32_results_are_not_biased_towards_zero(lib, prec, K):
    """Squared ReLU doubles what truncation takes from every sum."""
    c = Call(lib, 2000, 1858, K, 16, 1, 20, prec, act=oracle.ACT_RELU_2, out_f32=1, bias=False, ids=torch.full((2000,), -1))
    c.run()
    want = c.want()[0]
    assert abs(((c.out.double() - want).sum() / want.sum()).item()) <= 2 * rounded(0)


@gpu
@pytest.mark.parametrize("prec", [1, 2])
@pytest.mark.parametrize("M,N,group", [(500, 264, 1), (1500, 1000, 1), (1984, 520, 64)])
@pytest.mark.parametrize("K,rank", [(264, 16), (328, 16), (576, 48), (2056, 8), (2112, 128), (4104, 16), (8200, 32)])
def test_fp32_results_with_chains_that_end_early(lib, prec, M, N, group, K, rank):
    c = Call(lib, M, N, K, rank, group, 9, prec, out_f32=1)
    c.run()
    c.check()


@gpu
@pytest.mark.parametrize("prec", [0, 1, 2])
@pytest.mark.parametrize("pads,shift", [((8, 8, 8), 0), ((1, 3, 5), 0), ((8, 8, 8), 8), ((8, 8, 8), 1), ((0, 0, 1), 0), ((0, 8, 0), 3)])
@pytest.mark.parametrize("M,N,K,group", [(70, 72, 96, 1), (6400, 512, 256, 64)])
def test_strides_and_alignment(lib, prec, pads, shift, M, N, K, group):
    c = Call(lib, M, N, K, 16, group, 6, prec, pads=pads, shift=shift, bias=False, scales=False)
    c.run()
    c.check()


@gpu
@pytest.mark.parametrize("prec", [0, 1, 2])
@pytest.mark.parametrize("M,group", [(50, 1), (8192, 64)])
def test_requests_without_an_adapter(lib, prec, M, group):
    """Ids outside the adapters: the plain product, whatever the adapters hold."""
    requests = (M + group - 1) // group
    ids = torch.tensor([-1, 4, 0, -2147483648, 2147483647, 1] * requests)[:requests]
    c = Call(lib, M, 512, 256, 16, group, 4, prec, ids=ids)
    c.run()
    c.ids[c.ids > 3] = -1  # the same thing
    c.check()
    c.a[2:], c.b[2:], c.scales[2:] = float("nan"), float("nan"), float("inf")  # adapters that no request names
    first = c.run().clone()
    none = (c.ids.repeat_interleave(group)[:M] < 0)
    c.ids[:] = -1
    assert torch.equal(c.run()[none], first[none])
    c.check()


@gpu
def test_values_that_are_not_finite_stay_with_their_rows(lib):
    for M, group in ((40, 1), (8192, 64)):
        c = Call(lib, M, 512, 256, 16, group, 8, 2, ids=torch.arange((M + group - 1) // group) % 8)
        c.run()
        want, allowed = c.want()
        c.x[3, 5] = float("inf")
        c.b[5, 7, 2] = float("nan")
        c.a[6, 3] = float("inf")
        got = c.run()
        ids = c.ids.repeat_interleave(group)[:M]
        bad = torch.zeros(M, 512, dtype=torch.bool, device="cuda")
        bad[3] = True
        bad[ids == 6] = True
        bad[ids == 5, 7] = True
        # not the same bits: an element that the tensor core met as zero times NaN is summed again in another order, and each order is
        # within the allowance of the exact sum
        assert ((got.double() - want).abs() <= allowed)[~bad].all()
        assert not torch.isfinite(got[ids == 5, 7]).any() and not torch.isfinite(got[3]).any() and not torch.isfinite(got[ids == 6]).any()


@gpu
@pytest.mark.parametrize("M,group", [(40, 1), (1536, 64), (8192, 64)])
def test_narrow_products_beyond_the_range_of_fp16(lib, M, group):
    """X A^T up to 1e6 met by a small B: results of order one."""
    c = Call(lib, M, 512, 256, 16, group, 8, 1)
    c.a *= 2e4
    c.b *= 1e-5
    c.a[3] *= 1e-3  # one adapter whose products fit
    c.run()
    assert (c.x.float() @ c.a[0].float().T).abs().max() > 65504
    c.check()



BODIES = [(1536, 512, 256, 16, 64), (64, 256, 1024, 16, 64), (320, 512, 640, 40, 64),  # cut over clusters, X A^T row by row among them
          (8192, 512, 256, 16, 64), (32768, 1024, 128, 16, 64), (32768, 1024, 128, 32, 128), (24000, 1096, 192, 48, 64), (32768, 768, 128, 128, 192)]


@gpu
@pytest.mark.parametrize("a,b", [(1.0, 1.0), (1e-4, 1e4), (1e-5, 2e4), (3e-3, 300.0)])
@pytest.mark.parametrize("M,N,K,rank,group", BODIES)
def test_small_narrow_products_met_by_a_large_b(lib, M, N, K, rank, group, a, b):
    """X A^T far below what one fp16 value resolves, results of order one: as exact as the exact results rounded to fp16.  Sums in fp32
    (K / 8 truncated additions at most: 2^-20 here) add less than a hundredth to the rounding's 2^-12."""
    c = Call(lib, M, N, K, rank, group, 9, 1, ids=torch.randint(-1, 9, ((M + group - 1) // group,), generator=torch.Generator().manual_seed(M)))
    c.scales *= a  # the scale is in X A^T
    c.b *= b
    c.run()
    want, _ = c.want()
    with_one = (c.ids.repeat_interleave(group)[:M] >= 0)
    rms = lambda v: ((v.double() - want)[with_one].norm() / want[with_one].norm()).item()
    assert rms(c.out) <= 1.02 * rms(want.half()), (rms(c.out), rms(want.half()))
    # every element: half a step of the type, sums in fp32, of X A^T 22 bits or 2^-36 through B
    ids = c.ids.long().repeat_interleave(group)[:M]
    x, w = c.x.double(), c.w.double()
    err = x.abs() @ w.abs().T + c.bias.double().abs() + want.abs()
    err *= (K / 8 + 24) * 2.0 ** -24
    for j in range(9):
        r = (ids == j).nonzero()[:, 0]
        h, hmag = c.scales[j].double() * (x[r] @ c.a[j].double().T), c.scales[j].double() * (x[r].abs() @ c.a[j].double().abs().T)
        err[r] += (2.0 ** -22 * h.abs() + (K / 8 + 24) * 2.0 ** -24 * hmag + 2.0 ** -36) @ c.b[j].double().abs().T
    assert ((c.out.double() - want).abs() <= 2.0 ** -11 * want.abs() + (1 + 2.0 ** -11) * err + 2.0 ** -25).all()


@gpu
@pytest.mark.parametrize("M,N,K,rank,group", BODIES)
def test_large_narrow_products_met_by_a_small_b(lib, M, N, K, rank, group):
    """X A^T beyond fp16 in every kernel that makes or takes its two values."""
    c = Call(lib, M, N, K, rank, group, 8, 1)
    c.a *= 2e4
    c.b *= 1e-5
    c.a[3] *= 1e-3  # one adapter whose products fit
    c.run()
    if M > 64:  # (the one request of 64 rows may have none, or one whose products fit)
        assert max((c.x.float() @ c.a[j].float().T).abs().max() * c.scales[j] for j in set(c.ids.tolist()) - {-1}) > 65504
    c.check()
    c.ids[:] = -1
    plain = c.run().clone()
    c.ids[0] = 4  # rows beside a request whose pieces are infinite
    assert torch.equal(c.run()[group:], plain[group:])
    c.check()



@gpu
@pytest.mark.parametrize("M,N,K,rank,group", [(1536, 512, 256, 16, 64), (8192, 512, 256, 16, 64), (32768, 1024, 128, 16, 64), (32768, 768, 128, 32, 64),
                                              (24000, 1096, 192, 48, 64)])
def test_fp16_values_that_are_not_finite_stay_with_their_rows(lib, M, N, K, rank, group):
    c = Call(lib, M, N, K, rank, group, 8, 1, ids=torch.arange((M + group - 1) // group) % 9 - 1)
    c.run()
    want, allowed = c.want()
    c.x[3, 5] = float("inf")
    c.x[700, 1] = float("nan")
    c.b[5, 7, 2] = float("nan")
    c.b[2, 300, 1] = float("inf")
    c.a[6, 3] = float("inf")
    got = c.run()
    ids = c.ids.repeat_interleave(group)[:M]
    bad = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    bad[3], bad[700], bad[ids == 6] = True, True, True
    bad[ids == 5, 7] = True
    bad[ids == 2, 300] = True
    assert ((got.double() - want).abs() <= allowed)[~bad].all()  # (in another order of sums: each is within the allowance)
    assert not (got[bad].abs() < 65504).any()  # (an infinite result of fp16 is its largest number, as in b200_op_gemm)



@gpu
@pytest.mark.parametrize("prec", [1, 2])
@pytest.mark.parametrize("M,N,K,rank,group", [(1, 8, 8, 1, 1), (1, 1858, 64, 8, 1), (3, 130, 72, 5, 1), (64, 8, 128, 16, 64), (65, 136, 192, 24, 64),
                                              (129, 33, 8, 128, 64), (700, 40, 520, 12, 64), (10, 24, 4096, 16, 1), (2000, 72, 1000, 7, 30)])
def test_fp32_results_of_small_and_odd_shapes(lib, prec, M, N, K, rank, group):
    c = Call(lib, M, N, K, rank, group, 3, prec, out_f32=1, pads=(8, 0, 3))
    c.run()
    c.check()


@gpu
@pytest.mark.parametrize("prec", [1, 2])
@pytest.mark.parametrize("M,N,K,rank,group", [(32700, 1024, 128, 16, 64), (32513, 1024, 64, 32, 64), (19010, 1536, 72, 72, 64), (25001, 776, 136, 16, 192),
                                              (32768 + 64, 2048, 64, 8, 64), (600, 4872, 64, 16, 64)])
def test_bodies_whose_last_request_is_not_whole(lib, prec, M, N, K, rank, group):
    """Several tiles to a pair of CTAs, the last one with rows that are not there; one tile to a pair."""
    for adapters in (2, 40):  # requests of a tile that share an adapter, and not
        c = Call(lib, M, N, K, rank, group, adapters, prec)
        c.run()
        c.check()


@gpu
def test_captured_call_follows_the_ids(lib):
    c = Call(lib, 8192, 512, 256, 16, 64, 5, 1)
    s = torch.cuda.Stream()
    c.run(s.cuda_stream)
    c.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _lib.check(lib.b200_op_gemm_adapters(ctypes.byref(c.d), torch.cuda.current_stream().cuda_stream))
    for seed in range(3):
        c.ids.copy_(torch.randint(-1, 5, c.ids.shape, generator=torch.Generator().manual_seed(seed)))
        c.x.normal_()
        c.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        c.check()


@gpu
def test_two_calls_at_once(lib):
    """Two streams, a workspace each."""
    a, b = Call(lib, 16384, 1024, 512, 16, 64, 40, 1, seed=1), Call(lib, 1000, 512, 1024, 8, 1, 40, 2, seed=2)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        _lib.check(lib.b200_op_gemm_adapters(ctypes.byref(a.d), sa.cuda_stream))
        _lib.check(lib.b200_op_gemm_adapters(ctypes.byref(b.d), sb.cuda_stream))
    torch.cuda.synchronize()
    a.check()
    b.check()



@gpu
def test_calls_of_every_kind_at_once(lib):
    """A stream and a workspace each: the kernels of one call hold tensor memory, form clusters and wait for their H beside those of the others."""
    kinds = [(16384, 1024, 512, 16, 64, 1, 0), (2048, 1536, 512, 32, 64, 1, 0), (320, 512, 1024, 16, 64, 1, 0), (37, 1858, 2048, 16, 1, 2, 1),
             (1000, 264, 2048, 13, 1, 1, 0), (4096, 512, 1024, 128, 64, 2, 1), (1024, 512, 1536, 16, 64, 0, 0), (64, 256, 2048, 8, 64, 2, 0)]
    calls = [Call(lib, M, N, K, rank, group, 20, prec, out_f32=f32, seed=i) for i, (M, N, K, rank, group, prec, f32) in enumerate(kinds)]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, s in zip(calls, streams):
            _lib.check(lib.b200_op_gemm_adapters(ctypes.byref(c.d), s.cuda_stream))
    torch.cuda.synchronize()
    for c in calls:
        assert c.status.item() == 0
        c.check()


@gpu
def test_a_move_per_game_from_its_own_adapter(lib):
    """As a server of many games runs them: a shared policy head with an adapter per game, then a legal move from its logits."""
    from test_gpu_sample import draw, reference
    games = 75
    c = Call(lib, games, 1858, 2048, 16, 1, 20, 1, out_f32=1)
    g = torch.Generator().manual_seed(5)
    moves = torch.stack([torch.randperm(1858, generator=g)[:256] for _ in range(games)]).to(torch.int32).to(torch.uint16)
    counts = torch.randint(1, 60, (games,), generator=g).int()
    u, T, p = torch.rand(games, generator=g).numpy(), np.full(games, 0.8, np.float32), np.full(games, 0.95, np.float32)
    s = torch.cuda.Stream()
    logits = c.run(s.cuda_stream)
    c.check()
    choice, prob = draw(lib, logits, u, moves=moves.cuda(), counts=counts.cuda(), stream=s.cuda_stream, temperature=T, top_p=p)
    for i in range(games):
        l = logits[i].double().cpu().numpy()[moves[i, :counts[i]].numpy().astype(np.int64)]
        want = reference(l, T[i], 0, p[i], 0.0, u[i])
        assert choice[i] == want[0] and abs(prob[i] - want[1]) <= 80 * 2.0 ** -24


def test_refusals():
    lib = _lib.load()
    ok = dict(X=4096, W=4096, C=4096, A=4096, B=4096, ids=4096, M=64, N=64, K=64, activation=3, precision=1, n_adapters=2, rank=8,
              group=64, workspace=4096)
    need = ctypes.c_size_t()

    def both(**change):
        d = _lib.AdaptersDesc(**dict(ok, **change))
        size = lib.b200_op_gemm_adapters_workspace(ctypes.byref(d), ctypes.byref(need))
        if "workspace_bytes" not in change:
            d.workspace_bytes = need.value
        return size, lib.b200_op_gemm_adapters(ctypes.byref(d), None)

    assert lib.b200_op_gemm_adapters(None, None) == lib.b200_op_gemm_adapters_workspace(None, ctypes.byref(need)) == _lib.ERR_INVALID
    d = _lib.AdaptersDesc(**ok)
    assert lib.b200_op_gemm_adapters_workspace(ctypes.byref(d), None) == _lib.ERR_INVALID
    for change in (dict(M=-1), dict(M=64 * 65535 + 1), dict(N=0), dict(K=0), dict(rank=0), dict(rank=129), dict(n_adapters=0), dict(group=0), dict(precision=3),
                   dict(activation=0), dict(activation=9), dict(ldx=63), dict(ldw=8), dict(ldc=63), dict(ldc=-64)):
        assert both(**change) == (_lib.ERR_INVALID, _lib.ERR_INVALID), change
        assert b"b200_op_gemm_adapters" in lib.b200_last_error()
    for change in (dict(X=None), dict(W=None), dict(C=None), dict(A=None), dict(B=None), dict(ids=None), dict(workspace=None),
                   dict(workspace=4096 + 128), dict(workspace_bytes=16), dict(X=4097), dict(bias=4098), dict(C=4098, out_f32=1),
                   dict(ids=4098), dict(scales=4097), dict(status=4098)):
        assert both(**change) == (_lib.OK, _lib.ERR_INVALID), change
    assert both(M=0, X=None, W=None, C=None, A=None, B=None, ids=None, workspace=None) == (_lib.OK, _lib.OK)


@pytest.mark.parametrize("prec", [0, 1, 2])
@pytest.mark.parametrize("out_f32", [0, 1])
@pytest.mark.parametrize("M,N,K,rank,group", [(1, 8, 8, 1, 1), (1024, 512, 256, 16, 1), (1024, 512, 256, 16, 64), (64, 512, 256, 16, 64), (63, 512, 256, 16, 1),
                                              (1000, 500, 252, 13, 7), (8192, 1024, 1024, 64, 64), (4096, 1858, 2048, 32, 1)])
def test_workspace_of_a_description_without_pointers(prec, out_f32, M, N, K, rank, group):
    """The size asked for before the tensors exist is that of the call with them."""
    lib = _lib.load()
    sizes = []
    for pointers in ({}, dict(X=4096, W=8192, C=12288, A=4096, B=4096, ids=4096, bias=4096, scales=4096)):
        d = _lib.AdaptersDesc(M=M, N=N, K=K, activation=oracle.ACT_NONE, precision=prec, out_f32=out_f32, n_adapters=5, rank=rank, group=group, **pointers)
        need = ctypes.c_size_t()
        assert lib.b200_op_gemm_adapters_workspace(ctypes.byref(d), ctypes.byref(need)) == _lib.OK
        sizes.append(need.value)
    assert sizes[0] == sizes[1]
