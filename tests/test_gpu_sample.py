"""b200_op_sample against numpy in 64 bits: the same entry for every row, its probability in fp32."""
import ctypes

import numpy as np
import pytest

from lc0_b200 import _lib

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

DT = {0: torch.float32, 1: torch.float16, 2: torch.bfloat16}
INF = float("inf")


def reference(l, T=1.0, k=0, p=1.0, min_p=0.0, u=0.0):
    """(choice, probability) of one row of float64 logits; the numbers are the float32 ones the operator gets."""
    T, p, min_p, u = (float(np.float32(x)) for x in (T, p, min_p, u))
    l = np.where(np.isnan(l), -INF, l)
    if not (l > -INF).any():
        return -1, 0.0
    top = l.max()
    if not T > 0:
        return int(np.argmax(l == top)), 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(l == top, 1.0, 0.0 if top == INF else np.exp((l - top) / T))
    order = [i for i in np.argsort(-l, kind="stable") if l[i] > -INF]
    if k > 0:
        order = order[:k]
    if p < 1:
        mass = np.concatenate([[0.0], np.cumsum(w[order])])
        order = order[:max(1, int((mass[:-1] < p * mass[-1]).sum()))]
    if min_p > 0:
        order = [i for i in order if w[i] >= min(min_p, 1.0)]
    kept = np.sort(order)
    mass = np.cumsum(w[kept])
    u = min(u, 1 - 2.0 ** -24) if u >= 0 else 0.0
    at = kept[int(np.argmax(mass > u * mass[-1]))]
    return int(at), float(w[at] / mass[-1])


def draw(lib, logits, u, moves=None, counts=None, stream=None, **per_row):
    """The operator on CUDA tensors; per_row: temperature, top_k, top_p, min_p as sequences or None."""
    rows = logits.shape[0]
    choice = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    prob = torch.full((rows,), -7.0, device="cuda")
    held = dict(u=torch.as_tensor(np.asarray(u, np.float32)).cuda())
    for name, v in per_row.items():
        if v is not None:
            held[name] = torch.as_tensor(np.asarray(v, np.int32 if name == "top_k" else np.float32)).cuda()
    d = _lib.SampleDesc(logits=logits.data_ptr(), ld=logits.stride(0) if rows > 1 else 0, rows=rows, width=logits.shape[1],
                        precision={v: k for k, v in DT.items()}[logits.dtype], choice=choice.data_ptr(), prob=prob.data_ptr(),
                        **{n: v.data_ptr() for n, v in held.items()})
    if moves is not None:
        d.move_ids, d.n_moves, d.ld_moves = moves.data_ptr(), counts.data_ptr(), moves.shape[1]
    torch.cuda.synchronize()  # the inputs are made on another stream
    _lib.check(lib.b200_op_sample(ctypes.byref(d), stream))
    torch.cuda.synchronize()
    return choice.cpu().numpy(), prob.cpu().numpy()


def compare(rows, got, u, T=None, k=None, p=None, min_p=None):
    choice, prob = got
    at = lambda v, i, off: off if v is None else v[i]
    for i, l in enumerate(rows):
        want = reference(l, at(T, i, 1.0), at(k, i, 0), at(p, i, 1.0), at(min_p, i, 0.0), u[i])
        assert choice[i] == want[0], (i, choice[i], want, prob[i])
        # weights: the difference to the largest logit, rounded once, is an exponent of up to |z| = 20 where the weight counts; exp2f 2
        # steps; chains of up to 4 * 13 additions; the result's rounding
        assert abs(prob[i] - want[1]) <= (20 + 4 + 52 + 1) * 2.0 ** -24 * want[1] + 1e-37, (i, prob[i], want)


def settings(rng, rows, kind):
    T = rng.uniform(0.2, 2.0, rows).astype(np.float32) if kind != "plain" else None
    k = rng.integers(0, 70, rows).astype(np.int32) if kind in ("k", "all") else None
    p = rng.uniform(0.2, 1.1, rows).astype(np.float32) if kind in ("p", "all") else None
    m = rng.uniform(0, 0.2, rows).astype(np.float32) if kind in ("min", "all") else None
    return T, k, p, m


@gpu
@pytest.mark.parametrize("kind", ["plain", "k", "p", "min", "all"])
@pytest.mark.parametrize("rows,width", [(3, 1), (5, 2), (33, 31), (7, 32), (4, 33), (9, 128), (65, 511), (3, 513), (150, 1858),
                                        (1, 1858), (6, 2049), (5, 4288), (3, 8192), (3, 8193), (2, 53248), (2, 60001), (1, 262144)])
def test_rows(lib, kind, rows, width):
    rng = np.random.default_rng(rows * 7 + width)
    prec = int(rng.integers(0, 3))
    pad, shift = int(rng.integers(0, 6)), int(rng.integers(0, 5))
    held = torch.from_numpy((rng.standard_normal((rows, width + pad)) * 3).astype(np.float32)).to(DT[prec])
    flat = torch.empty(shift + held.numel(), dtype=DT[prec], device="cuda")  # rows on any boundary of their type
    flat[shift:] = held.flatten().cuda()
    logits = flat[shift:].view(rows, width + pad)[:, :width]
    T, k, p, m = settings(rng, rows, kind)
    u = rng.random(rows, np.float32)
    got = draw(lib, logits, u, temperature=T, top_k=k, top_p=p, min_p=m)
    compare(held[:, :width].double().numpy(), got, u, T, k, p, m)


@gpu
@pytest.mark.parametrize("prec", [0, 1, 2])
@pytest.mark.parametrize("spread", [0.0, 0.5, 3.0, 40.0])
@pytest.mark.parametrize("width", [218, 1858])
def test_ties_and_spreads(lib, prec, spread, width):
    """Logits on a coarse grid: cuts inside runs of equal entries; flat rows, whose thresholds lie closest together."""
    rng = np.random.default_rng(int(spread * 10) + width)
    rows = 400
    held = torch.from_numpy(np.round(rng.standard_normal((rows, width)) * spread * 2).astype(np.float32) / 2).to(DT[prec])
    T, k, p, m = settings(rng, rows, "all")
    k[::3], p[1::3] = 0, 1.0
    u = rng.random(rows, np.float32)
    got = draw(lib, held.cuda(), u, temperature=T, top_k=k, top_p=p, min_p=m)
    compare(held.double().numpy(), got, u, T, k, p, m)


@gpu
@pytest.mark.parametrize("width", [8, 256, 2048, 16384, 65536])
def test_thresholds_that_are_met_exactly(lib, width):
    """Equal weights: u and top_p fall on sums themselves, where one rounding either way is another entry."""
    rng = np.random.default_rng(width)
    rows = 32
    u = (rng.integers(0, min(width, 1 << 20), rows) / width).astype(np.float32)
    p = (rng.integers(1, width, rows) / width).astype(np.float32)
    u[0], u[1], p[2] = 0.0, 1.0, 1.0 / width
    held = np.zeros((rows, width), np.float32)
    compare(held, draw(lib, torch.from_numpy(held).cuda(), u), u)
    compare(held, draw(lib, torch.from_numpy(held).cuda(), u, top_p=p), u, p=p)


@gpu
@pytest.mark.parametrize("prec", [0, 1, 2])
@pytest.mark.parametrize("width", [40, 700, 9000])
def test_masks_and_extreme_values(lib, prec, width):
    low = float(torch.finfo(DT[prec]).min)
    rng = np.random.default_rng(width)
    held = torch.from_numpy(rng.standard_normal((16, width)).astype(np.float32)).to(DT[prec])
    held[0] = -INF                       # nothing left
    held[1] = float("nan")
    held[2] = low                        # all at the lowest value: equal weights
    held[3] = low
    held[3, 17] = 0.5                    # one entry beside a mask of lowest values
    held[4] = -INF
    held[4, width - 1] = low             # one entry left, the lowest value
    held[5, ::2], held[5, 1::4] = -INF, float("nan")
    held[6, 3], held[6, 30] = INF, INF   # infinities share
    held[7] = -float(torch.finfo(DT[prec]).max)
    held[7, 5] = float(torch.finfo(DT[prec]).max)
    held[8, 0] = -0.0
    held[8, 1:] = -0.0
    held[8, 9] = 0.0                     # one key for both zeros
    held[9] *= 1e-3 if prec else 1e-30
    u = rng.random(16, np.float32)
    T = np.full(16, 0.7, np.float32)
    T[10], T[11], T[12], T[13], T[7], T[14] = 0.0, -1.0, float("nan"), 1e-40, 3e38, 1e6
    rows = held.double().numpy()
    compare(rows, draw(lib, held.cuda(), u, temperature=T), u, T=T)
    k = rng.integers(1, 6, 16).astype(np.int32)
    compare(rows, draw(lib, held.cuda(), u, temperature=T, top_k=k), u, T=T, k=k)
    p = np.full(16, 0.4, np.float32)
    p[3:6] = 0.0, -2.0, float("nan")
    compare(rows, draw(lib, held.cuda(), u, temperature=T, top_p=p), u, T=T, p=p)
    m = np.full(16, 0.5, np.float32)
    m[:3] = 1.0, 2.0, float("nan")
    compare(rows, draw(lib, held.cuda(), u, temperature=T, min_p=m), u, T=T, min_p=m)


@gpu
def test_random_numbers_at_their_ends(lib):
    rng = np.random.default_rng(3)
    held = (rng.standard_normal((8, 300)) * 60).astype(np.float32)  # most weights are zero in 32 bits
    u = np.array([0.0, 1 - 2.0 ** -24, 1.0, 7.0, -3.0, np.nan, 1e-30, 2.0 ** -24], np.float32)
    compare(held.astype(np.float64), draw(lib, torch.from_numpy(held).cuda(), u), u)


@gpu
@pytest.mark.parametrize("prec", [0, 1, 2])
@pytest.mark.parametrize("rows,ld_moves", [(1, 256), (97, 256), (3, 1), (2, 1900)])
def test_lists_of_moves(lib, prec, rows, ld_moves):
    """Entries by index, lists of any length up to the stride, the same entry twice, indices outside the row."""
    rng = np.random.default_rng(rows + ld_moves)
    held = torch.from_numpy((rng.standard_normal((rows, 1858)) * 2).astype(np.float32)).to(DT[prec])
    ids = rng.integers(0, 1858, (rows, ld_moves)).astype(np.uint16)
    ids[:, 0] = 1857
    if ld_moves > 8:
        ids[:, 5] = ids[:, 2]
        ids[:, 7], ids[:, 6] = 1858, 65535
    counts = rng.integers(0, ld_moves + 1, rows).astype(np.int32)
    if rows > 4:
        counts[:4] = 0, -5, ld_moves + 100, 1
    T, k, p, m = settings(rng, rows, "all")
    u = rng.random(rows, np.float32)
    got = draw(lib, held.cuda(), u, moves=torch.from_numpy(ids).cuda(), counts=torch.from_numpy(counts).cuda(), temperature=T, top_k=k,
               top_p=p, min_p=m)
    lists = []
    for i in range(rows):
        j = ids[i, :min(max(counts[i], 0), ld_moves)].astype(np.int64)
        lists.append(np.where(j < 1858, held[i].double().numpy()[np.minimum(j, 1857)], -INF))
        if not lists[-1].size:
            lists[-1] = np.array([-INF])
    compare(lists, got, u, T, k, p, m)


@gpu
def test_lists_of_entries_of_wide_rows(lib):
    """Indices are 16 bits: a list names entries among the first 65536 of a wider row and nothing else."""
    rng = np.random.default_rng(9)
    held = rng.standard_normal((5, 70000)).astype(np.float32)
    held[:, 65536:] += 50  # never named
    ids = rng.integers(0, 65536, (5, 300)).astype(np.uint16)
    counts = np.array([300, 3, 70, 0, 256], np.int32)
    u = rng.random(5, np.float32)
    got = draw(lib, torch.from_numpy(held).cuda(), u, moves=torch.from_numpy(ids).cuda(), counts=torch.from_numpy(counts).cuda())
    compare([held[i].astype(np.float64)[ids[i, :c]] if c else np.array([-INF]) for i, c in enumerate(counts)], got, u)


@gpu
@pytest.mark.parametrize("temperature", [1e-44, 1e-37, 1e-20, 1e29, 1e31, 3e38, INF])
def test_temperatures_of_every_size(lib, temperature):
    rng = np.random.default_rng(4)
    held = (rng.standard_normal((20, 700)) * 1e3).astype(np.float32)
    u, T, p = rng.random(20, np.float32), np.full(20, temperature, np.float32), np.full(20, 0.5, np.float32)
    compare(held.astype(np.float64), draw(lib, torch.from_numpy(held).cuda(), u, temperature=T), u, T=T)
    compare(held.astype(np.float64), draw(lib, torch.from_numpy(held).cuda(), u, temperature=T, top_p=p), u, T=T, p=p)


@gpu
def test_a_row_does_not_depend_on_its_batch_or_stream(lib):
    g = torch.Generator(device="cuda").manual_seed(1)
    logits, u = torch.randn(2000, 1858, device="cuda", generator=g) * 3, torch.rand(2000, generator=torch.Generator().manual_seed(2)).numpy()
    p = np.full(2000, 0.9, np.float32)
    whole = draw(lib, logits, u, top_p=p)
    s = torch.cuda.Stream()
    for n in (1, 2, 37, 300):
        part = draw(lib, logits[5:5 + n], u[5:5 + n], top_p=p[:n], stream=s.cuda_stream)
        assert np.array_equal(part[0], whole[0][5:5 + n])
        assert np.allclose(part[1], whole[1][5:5 + n], rtol=80 * 2.0 ** -24, atol=0)



@gpu
@pytest.mark.parametrize("grid", [0, 8])
def test_rows_of_warps_that_gather_unevenly(lib, grid):
    """The end of top-p among entries that the lanes of a warp put side by side, some lanes many, most none: logits fall over the row,
    so that the heavy ones are one lane's.  The same answer every time."""
    rng = np.random.default_rng(grid)
    rows, width = 2000, 1200
    held = rng.standard_normal((rows, width)) - np.linspace(0, 12, width) * rng.uniform(0, 1, (rows, 1))
    held = (np.round(held * grid) / grid if grid else held).astype(np.float32)
    u, p = rng.random(rows, np.float32), rng.uniform(0.05, 0.99, rows).astype(np.float32)
    logits = torch.from_numpy(held).cuda()
    first = draw(lib, logits, u, top_p=p)
    compare(held.astype(np.float64), first, u, p=p)
    for _ in range(4):
        again = draw(lib, logits, u, top_p=p)
        assert np.array_equal(again[0], first[0]) and np.array_equal(again[1], first[1])



@gpu
@pytest.mark.parametrize("kind", ["plain", "k", "p", "all"])
@pytest.mark.parametrize("rows,width", [(1, 262144), (40, 20000), (150, 50257)])
def test_waits_that_give_up(lib, kind, rows, width):
    """One CTA of a cluster gives up at any of its waits, the others wait for it in vain: the launch ends, and a row has its answer (where
    that CTA has fewer waits) or -2 and 0."""
    rng = np.random.default_rng(rows)
    held = torch.from_numpy((rng.standard_normal((rows, width)) * 2).astype(np.float32)).to(torch.bfloat16)
    logits = held.cuda()
    T, k, p, m = settings(rng, rows, kind)
    if kind == "k":
        k = rng.integers(1, width, rows).astype(np.int32)
    u = rng.random(rows, np.float32)
    call = lambda: draw(lib, logits, u, temperature=T, top_k=k, top_p=p, min_p=m)
    right = call()
    at = sorted(rng.choice(rows, min(rows, 5), replace=False))
    one = lambda v: None if v is None else v[at]
    compare(held[at].double().numpy(), (right[0][at], right[1][at]), u[at], one(T), one(k), one(p), one(m))
    gave_up = []
    try:
        for wait in range(14):
            lib.b200_op_sample_inject_give_up(wait * 5 % (2 if width < 50000 else 4), wait)
            choice, prob = call()
            out = choice == -2
            gave_up.append(int(out.sum()))
            assert (prob[out] == 0).all()
            assert np.array_equal(choice[~out], right[0][~out]) and np.array_equal(prob[~out], right[1][~out]), wait
    finally:
        lib.b200_op_sample_inject_give_up(-1, -1)
    assert gave_up[0] == rows and gave_up == sorted(gave_up, reverse=True), gave_up
    again = call()
    assert np.array_equal(again[0], right[0]) and np.array_equal(again[1], right[1])



@gpu
def test_a_move_from_the_policy_that_a_network_leaves_on_the_device(lib):
    """b200_net_enqueue_device, then the draw on b200_net_stream: nothing in between goes over the host."""
    from conftest import load_case
    from lc0_b200 import network
    net, pos, n, _ = load_case("cfg4_mini")
    n = min(n, 16)
    nw = network.Network(net, "precision=fp16,max_batch=16")
    masks = torch.from_numpy(pos["masks"][:n].astype(np.int64)).cuda()
    values = torch.from_numpy(pos["values"][:n].astype(np.float32)).cuda()
    policy, qdm = torch.zeros(n, 1858, device="cuda"), torch.zeros(n, 3, device="cuda")
    rng = np.random.default_rng(6)
    moves = np.stack([rng.permutation(1858)[:256] for _ in range(n)]).astype(np.uint16)
    counts = rng.integers(1, 60, n).astype(np.int32)
    u, T = rng.random(n, np.float32), rng.uniform(0.3, 1.5, n).astype(np.float32)
    held = [torch.from_numpy(v).cuda() for v in (u, T, counts)]
    ids = torch.from_numpy(moves).cuda()
    choice, prob = torch.full((n,), -7, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda")
    d = _lib.SampleDesc(logits=policy.data_ptr(), rows=n, width=1858, u=held[0].data_ptr(), temperature=held[1].data_ptr(), move_ids=ids.data_ptr(),
                        n_moves=held[2].data_ptr(), ld_moves=256, choice=choice.data_ptr(), prob=prob.data_ptr())
    torch.cuda.synchronize()
    nw.enqueue_device(masks.data_ptr(), values.data_ptr(), n, policy.data_ptr(), qdm.data_ptr())
    _lib.check(lib.b200_op_sample(ctypes.byref(d), nw.stream()))
    nw.sync()
    logits = policy.double().cpu().numpy()
    assert (logits != 0).any()
    compare([logits[i][moves[i, :c].astype(np.int64)] for i, c in enumerate(counts)], (choice.cpu().numpy(), prob.cpu().numpy()), u, T=T)
    nw.close()



@gpu
@pytest.mark.parametrize("kind", ["plain", "k", "p", "min", "all"])
@pytest.mark.parametrize("rows,width", [(40, 60), (500, 1858), (20, 1858), (20, 50257)])
def test_probabilities_are_as_near_as_documented(lib, kind, rows, width):
    """2^-20 of themselves: weights of fp32 are off by 3 (ex2), 1 (its factor) and |z|, on average at most ln n < 8, steps of 2^-24, their
    sums by 4; twice that is the bound of two sums compared, one of them is the total here."""
    rng = np.random.default_rng(rows + width)
    held = (rng.standard_normal((rows, width)) * 1.5).astype(np.float32)
    T, k, p, m = settings(rng, rows, kind)
    u = rng.random(rows, np.float32)
    choice, prob = draw(lib, torch.from_numpy(held).cuda(), u, temperature=T, top_k=k, top_p=p, min_p=m)
    at = lambda v, i, off: off if v is None else v[i]
    for i in range(rows):
        want = reference(held[i].astype(np.float64), at(T, i, 1.0), at(k, i, 0), at(p, i, 1.0), at(m, i, 0.0), u[i])
        assert choice[i] == want[0] and abs(prob[i] - want[1]) <= 2.0 ** -20 * want[1], (i, choice[i], prob[i], want)


@gpu
def test_captured_and_replayed(lib):
    logits, u = torch.randn(64, 1858, device="cuda"), torch.rand(64, device="cuda")
    choice, prob = torch.empty(64, dtype=torch.int32, device="cuda"), torch.empty(64, device="cuda")
    d = _lib.SampleDesc(logits=logits.data_ptr(), rows=64, width=1858, u=u.data_ptr(), choice=choice.data_ptr(), prob=prob.data_ptr())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _lib.check(lib.b200_op_sample(ctypes.byref(d), torch.cuda.current_stream().cuda_stream))
    for i in range(3):
        logits.copy_(torch.randn(64, 1858, device="cuda") * 3)
        u.copy_(torch.rand(64, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        compare(logits.double().cpu().numpy(), (choice.cpu().numpy(), prob.cpu().numpy()), u.cpu().numpy())


def test_refusals():
    lib = _lib.load()
    x = ctypes.c_void_p(4096)  # never reached
    ok = dict(logits=4096, rows=2, width=10, u=4096, choice=4096)

    def code(**change):
        d = _lib.SampleDesc(**dict(ok, **change))
        return lib.b200_op_sample(ctypes.byref(d), None)

    assert lib.b200_op_sample(None, None) == _lib.ERR_INVALID
    for change in (dict(rows=-1), dict(width=0), dict(width=262145), dict(precision=3), dict(precision=-1), dict(ld=9), dict(ld=-1),
                   dict(logits=None), dict(u=None), dict(choice=None), dict(logits=4098), dict(precision=1, logits=4097), dict(u=4098), dict(prob=4097),
                   dict(top_k=4098), dict(temperature=4099), dict(move_ids=4097, n_moves=4096, ld_moves=4),
                   dict(move_ids=x, ld_moves=4), dict(n_moves=x), dict(move_ids=x, n_moves=x, ld_moves=0),
                   dict(move_ids=x, n_moves=x, ld_moves=65537), dict(rows=1 << 30)):
        assert code(**change) == _lib.ERR_INVALID, change
        assert b"b200_op_sample" in lib.b200_last_error()
    assert code(rows=0, logits=None, u=None, choice=None) == _lib.OK
