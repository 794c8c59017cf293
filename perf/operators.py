"""The operators for batches that serve many games at once, as cases that can be timed and compared.

  adapters  b200_op_gemm_adapters: a layer shared by all requests, with a low-rank adapter (a player, a style) per request
            beside it: C = act(X W^T + bias + scale_a (X A_a^T) B_a^T).  A request is a position: 64 rows in a network's body,
            one row in its heads.
  sample    b200_op_sample: one move per game drawn from its policy logits with temperature, top-k, top-p and min-p and a
            given random number, over all columns or over a list of legal moves.

The plain form of `adapters` is computed in 32 bits and rounded once.  That of `sample` is computed in 64: the draw and the
top-p cut compare a running sum of up to tens of thousands of terms with a threshold.
"""
import ctypes
import math

import numpy as np
import torch

own = False

DTYPE = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
PREC = {"fp32": 0, "fp16": 1, "bf16": 2}
ACTS = {"mish": 1, "none": 3, "relu2": 8}


def listed():
    return [
        # One position at the root of a search, an encoder product of the BT4-class network: 64 rows, one adapter; latency.
        dict(name="adapt_root_fp16", op="adapters", type="fp16", rows=64, n=1024, k=1024, rank=16, group=64, adapters=8, act="none", f32=False),
        # A search's minibatch: 24 positions of several games, the FFN's first product with its activation.
        dict(name="adapt_search_24", op="adapters", type="fp16", rows=24 * 64, n=1536, k=1024, rank=16, group=64, adapters=24, act="relu2", f32=False),
        # The batch of the headline throughput, one adapter per position out of 256.
        dict(name="adapt_body_1024", op="adapters", type="fp16", rows=1024 * 64, n=1024, k=1024, rank=16, group=64, adapters=256, act="none", f32=False),
        # The other 16-bit type at a ragged batch and the largest rank; the FFN's second product.
        dict(name="adapt_body_333_bf16", op="adapters", type="bf16", rows=333 * 64, n=1024, k=1536, rank=64, group=64, adapters=40, act="none", f32=False),
        # A head's hidden layer, one row per position: value head of the BT4-class network over a throughput batch.
        dict(name="adapt_value_1024", op="adapters", type="fp16", rows=1024, n=128, k=2048, rank=8, group=1, adapters=64, act="mish", f32=False),
        # The classical policy head (32 planes x 64 squares -> 1858 logits in fp32), odd numbers of rows and columns.
        dict(name="adapt_policy_37", op="adapters", type="bf16", rows=37, n=1858, k=2048, rank=16, group=1, adapters=12, act="none", f32=True),
        # fp32 verification mode, the small attention network.
        dict(name="adapt_fp32_16", op="adapters", type="fp32", rows=16 * 64, n=512, k=256, rank=16, group=64, adapters=16, act="mish", f32=False),
        # One game's move: legal moves of one position, plain temperature; latency.
        dict(name="sample_move_1", op="sample", type="fp32", rows=1, n=1858, moves=True, top_k=False, top_p=False, min_p=False),
        # Selfplay with a thousand games: legal moves, every cut.
        dict(name="sample_moves_1024", op="sample", type="fp32", rows=1024, n=1858, moves=True, top_k=True, top_p=True, min_p=True),
        # Raw policies of a search's minibatch, top-p alone.
        dict(name="sample_policy_24", op="sample", type="fp16", rows=24, n=1858, moves=False, top_k=False, top_p=True, min_p=False),
        # Raw policies of large batches, every cut; the most data.
        dict(name="sample_policy_8192", op="sample", type="fp32", rows=8192, n=1858, moves=False, top_k=True, top_p=True, min_p=True),
        # Rows far wider than a policy, a few at a time.
        dict(name="sample_wide_48_bf16", op="sample", type="bf16", rows=48, n=50257, moves=False, top_k=False, top_p=True, min_p=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.55:
        kind = rng.choice(["body", "body", "head", "head", "fp32"])
        c = dict(op="adapters", type=rng.choice(["fp16", "bf16"]), act=rng.choice(["none", "mish", "relu2"]), f32=False)
        if kind == "head":
            c.update(rows=_log(rng, 1, 4096), n=rng.choice([32, 128, 256, 1000, 1858]), k=rng.choice([256, 512, 1024, 2048]),
                     group=1, rank=rng.choice([4, 8, 16, 32]), adapters=_log(rng, 1, 128), f32=rng.random() < 0.4)
        else:
            c.update(rows=64 * _log(rng, 1, 640), n=rng.choice([256, 512, 768, 1024, 1536]), k=rng.choice([256, 512, 1024, 1536]),
                     group=64 * rng.choice([1, 1, 1, 2, 3]), rank=rng.choice([8, 16, 24, 32, 64]), adapters=_log(rng, 1, 256))
        if kind == "fp32":
            c.update(type="fp32", rows=64 * _log(rng, 1, 48), rank=rng.choice([4, 8, 13, 16]))
        return c
    c = dict(op="sample", type=rng.choice(["fp32", "fp32", "fp16", "bf16"]), moves=False,
             top_k=rng.random() < 0.5, top_p=rng.random() < 0.6, min_p=rng.random() < 0.4)
    kind = rng.choice(["moves", "policy", "policy", "wide"])
    if kind == "moves":
        c.update(moves=True, n=1858, rows=_log(rng, 1, 8192))
    elif kind == "policy":
        c.update(n=rng.choice([1858, 1858, 4096, 4288, _log(rng, 2, 4096)]))
        c.update(rows=_log(rng, 1, 8192 * 1858 // max(c["n"], 1858)))
    else:
        c.update(n=_log(rng, 5000, 131072))
        c.update(rows=_log(rng, 1, max(1, 48 * 50257 // c["n"])))
    return c


def _inputs(case, seed):
    """The case's inputs from its seed.  Linear layers: activations of order one, weights of fan-in scale, adapters whose
    product is a fraction of the layer's; one request in eight has no adapter (id -1).  Policies: logits of a trained
    network's spread, of which a few stand out."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPE[case["type"]]

    def rnd(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "adapters":
        m, n, k, r, a = (case[x] for x in ("rows", "n", "k", "rank", "adapters"))
        d = dict(x=rnd(m, k).to(t), w=(rnd(n, k) * k ** -0.5).to(t), bias=rnd(n) * 0.1, a=(rnd(a, r, k) * k ** -0.5).to(t),
                 b=(rnd(a, n, r) * 0.4 * r ** -0.5).to(t), scales=0.5 + torch.rand(a, device="cuda", generator=g))
        requests = (m + case["group"] - 1) // case["group"]
        ids = torch.randint(0, a, (requests,), device="cuda", generator=g)
        d["ids"] = torch.where(torch.rand(requests, device="cuda", generator=g) < 0.125, -1, ids).int()
        return d
    rows, n = case["rows"], case["n"]
    logits = rnd(rows, n) * 1.5
    logits += 5.0 * (torch.rand(rows, n, device="cuda", generator=g) < min(1.0, 12.0 / n)) * torch.rand(rows, n, device="cuda", generator=g)
    d = dict(logits=logits.to(t), u=torch.rand(rows, device="cuda", generator=g),
             temperature=0.3 + 1.2 * torch.rand(rows, device="cuda", generator=g))
    if case["moves"]:
        count = (31 + 11 * rnd(rows)).round().clamp(1, 218).int()
        order = torch.rand(rows, n, device="cuda", generator=g).argsort(dim=1)[:, :256]
        d.update(moves=order.to(torch.int32).to(torch.uint16), n_moves=count)
    if case["top_k"]:
        d["top_k"] = torch.randint(1, 65, (rows,), device="cuda", generator=g).int()
    if case["top_p"]:
        d["top_p"] = 0.6 + 0.39 * torch.rand(rows, device="cuda", generator=g)
    if case["min_p"]:
        d["min_p"] = 0.1 * torch.rand(rows, device="cuda", generator=g)
    return d


def prepare(case, seed):
    s = dict(case=case, **_inputs(case, seed))
    torch.cuda.synchronize()
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------
def _activate(v, act):
    if act == "mish":
        return v * torch.tanh(torch.log1p(torch.exp(-v.abs())) + v.clamp(min=0))
    return v.clamp(min=0) ** 2 if act == "relu2" else v


def _adapters_plain(s):
    c = s["case"]
    m, group = c["rows"], c["group"]
    x = s["x"].float()
    y = x @ s["w"].float().T + s["bias"]
    requests = s["ids"].shape[0]
    none = (s["ids"] < 0) | (s["ids"] >= c["adapters"])
    ids = torch.where(none, 0, s["ids"]).long()
    scale = torch.where(none, 0.0, s["scales"][ids])
    a, b = s["a"].float(), s["b"].float()
    if m < requests * group:  # the last request has fewer rows
        x = torch.cat([x, x.new_zeros(requests * group - m, c["k"])])
    x = x.view(requests, group, c["k"])
    low = torch.empty(requests, group, c["n"], device=x.device)
    step = max(1, (1 << 28) // (c["rank"] * (c["k"] + c["n"])))  # the adapters of that many requests are gathered at a time
    for i in range(0, requests, step):
        j = ids[i:i + step]
        low[i:i + step] = (x[i:i + step] @ a[j].transpose(1, 2)) @ b[j].transpose(1, 2) * scale[i:i + step, None, None]
    y = _activate(y + low.view(requests * group, c["n"])[:m], c["act"])
    return y if c["f32"] else y.to(s["x"].dtype)


def _sample_plain(s):
    c = s["case"]
    if c["moves"]:
        at = torch.arange(256, device="cuda")
        l = torch.gather(s["logits"].double(), 1, s["moves"].long())
        l = torch.where(at < s["n_moves"][:, None], l, -math.inf)
    else:
        l = s["logits"].double()
    l = torch.where(l.isnan(), -math.inf, l)
    top = l.max(dim=1, keepdim=True).values
    w = torch.where(l == top, 1.0, torch.exp((l - top) / s["temperature"].double()[:, None]))
    w = torch.where(l == -math.inf, 0.0, w)
    keep = l > -math.inf
    if c["top_k"] or c["top_p"]:
        by_size = torch.sort(l, dim=1, descending=True, stable=True).indices
        ws = torch.gather(w, 1, by_size)
        kept = torch.gather(keep, 1, by_size)
        if c["top_k"]:
            kept &= torch.arange(l.shape[1], device="cuda") < s["top_k"][:, None]
            ws = torch.where(kept, ws, 0.0)
        if c["top_p"]:
            mass = torch.cumsum(ws, 1)
            before = mass - ws
            before[:, 0] = -1.0
            kept &= before < s["top_p"].double()[:, None] * mass[:, -1:]
        keep = torch.zeros_like(keep).scatter_(1, by_size, kept)
    if c["min_p"]:
        keep &= w >= s["min_p"].double()[:, None]
    w = torch.where(keep, w, 0.0)
    mass = torch.cumsum(w, 1)
    total = mass[:, -1:]
    hit = mass > s["u"].double()[:, None] * total
    choice = torch.where(hit.any(dim=1), hit.int().argmax(dim=1), -1)
    prob = torch.gather(w, 1, choice.clamp(min=0)[:, None]) / total
    return choice.int(), torch.where(choice >= 0, prob[:, 0], 0.0).float()


# ---- the framework's operators ----------------------------------------------------------------------------------
def _own(s):
    """Description of the call, outputs and workspace: made at a state's first pass and kept, as a program does."""
    from lc0_b200 import _lib
    lib, c = _lib.load(), s["case"]

    def p(name):
        return s[name].data_ptr() if name in s else None

    if c["op"] == "adapters":
        out = torch.empty(c["rows"], c["n"], device="cuda", dtype=torch.float32 if c["f32"] else s["x"].dtype)
        d = _lib.AdaptersDesc(X=p("x"), W=p("w"), bias=p("bias"), C=out.data_ptr(), M=c["rows"], N=c["n"], K=c["k"],
                              activation=ACTS[c["act"]], precision=PREC[c["type"]], out_f32=int(c["f32"]), A=p("a"), B=p("b"),
                              scales=p("scales"), n_adapters=c["adapters"], rank=c["rank"], ids=p("ids"), group=c["group"])
        need = ctypes.c_size_t()
        _lib.check(lib.b200_op_gemm_adapters_workspace(ctypes.byref(d), ctypes.byref(need)))
        work, status = torch.empty(need.value, dtype=torch.uint8, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        d.workspace, d.workspace_bytes, d.status = work.data_ptr(), need.value, status.data_ptr()
        return _lib.check, lib.b200_op_gemm_adapters, d, out, (work, status)
    choice = torch.empty(c["rows"], dtype=torch.int32, device="cuda")
    prob = torch.empty(c["rows"], dtype=torch.float32, device="cuda")
    d = _lib.SampleDesc(logits=p("logits"), rows=c["rows"], width=c["n"], precision=PREC[c["type"]], move_ids=p("moves"),
                        n_moves=p("n_moves"), ld_moves=256 if c["moves"] else 0, temperature=p("temperature"), top_k=p("top_k"),
                        top_p=p("top_p"), min_p=p("min_p"), u=p("u"), choice=choice.data_ptr(), prob=prob.data_ptr())
    return _lib.check, lib.b200_op_sample, d, (choice, prob), None


def run(s):
    if own:
        if "call" not in s:
            s["call"] = _own(s)
        check, op, d, out, _ = s["call"]
        check(op(ctypes.byref(d), torch.cuda.current_stream().cuda_stream))
        return out
    return _adapters_plain(s) if s["case"]["op"] == "adapters" else _sample_plain(s)


# ---- definitions in 64 bits -------------------------------------------------------------------------------------
def _adapters_exact(c, d):
    m, group = c["rows"], c["group"]
    out = torch.empty(m, c["n"], dtype=torch.float64, device="cuda")
    w, a, b = d["w"].double(), d["a"].double(), d["b"].double()
    of_row = d["ids"].repeat_interleave(group)[:m]
    for i in range(0, m, 8192):
        out[i:i + 8192] = torch.addmm(d["bias"].double(), d["x"][i:i + 8192].double(), w.T)
    for j in range(c["adapters"]):
        rows = (of_row == j).nonzero()[:, 0]
        out[rows] += (d["x"][rows].double() @ a[j].T @ b[j].T) * d["scales"][j].double()
    if c["act"] == "mish":
        out = out * torch.tanh(torch.logaddexp(out, torch.zeros_like(out)))
    elif c["act"] == "relu2":
        out = torch.relu(out).square()
    return out


def _sample_exact(c, d):
    h = {k: v.cpu() for k, v in d.items()}
    logits = h["logits"].double().numpy()
    choice, prob = np.full(c["rows"], -1, np.int32), np.zeros(c["rows"])
    for i in range(c["rows"]):
        l = logits[i]
        if c["moves"]:
            l = l[h["moves"][i, :int(h["n_moves"][i])].numpy().astype(np.int64)]
        w = np.exp((l - l.max()) / float(h["temperature"][i]))
        kept = np.ones(l.size, bool)
        if c["top_k"] or c["top_p"]:
            first = np.argsort(-l, kind="stable")
            size = min(l.size, int(h["top_k"][i])) if c["top_k"] else l.size
            if c["top_p"]:
                mass = np.concatenate([[0.0], np.cumsum(w[first[:size]])])
                size = max(1, int(np.searchsorted(mass[:-1], float(h["top_p"][i]) * mass[-1], side="left")))
            kept[first[size:]] = False
        if c["min_p"]:
            kept &= w >= float(h["min_p"][i])
        ids = np.flatnonzero(kept)
        mass = np.cumsum(w[ids])
        at = int(np.searchsorted(mass, float(h["u"][i]) * mass[-1], side="right"))
        choice[i], prob[i] = ids[at], w[ids[at]] / mass[-1]
    return torch.from_numpy(choice), torch.from_numpy(prob)


def exact(case, seed):
    d = _inputs(case, seed)
    return _adapters_exact(case, d) if case["op"] == "adapters" else _sample_exact(case, d)


# ---- work -------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "adapters":
        m, n, k, r = (case[x] for x in ("rows", "n", "k", "rank"))
        size = 4 if case["type"] == "fp32" else 2
        requests = (m + case["group"] - 1) // case["group"]
        used = case["adapters"] * (1 - (1 - 1 / case["adapters"]) ** (requests * 7 / 8))  # expected number of them in the batch
        return {"bytes": size * (m * k + n * k) + (4 if case["f32"] else size) * m * n + 4 * n + used * (size * r * (k + n) + 4) + 4 * requests,
                "flops": 2 * m * n * k + 2 * m * r * (k + n) * 7 / 8}
    size = 4 if case["type"] == "fp32" else 2
    entries = 31 if case["moves"] else case["n"]
    row = entries * (size + 2 if case["moves"] else size) + 4 * (2 + case["top_k"] + case["top_p"] + case["min_p"] + case["moves"]) + 8
    return {"bytes": case["rows"] * row, "flops": case["rows"] * entries * 8}
