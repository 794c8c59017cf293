"""The operators of an encoder layer served with 8-bit products, experts and normalised heads, as cases that can be timed and compared.

  int8     b200_op_quantize_rows, b200_op_gemm_int8: a layer in 8-bit integers.  The activations are quantised row by row (a scale per
           token) and meet weights with a scale per channel: C = act(sx sw (Q W^T) + bias) + res.
  experts  b200_op_gemm_experts: products grouped by expert with ragged sizes.  A request (a token, or the 64 rows of a position) has
           `top_k` experts; `up` goes from tokens to the slots sorted by expert, `down` from slots back to tokens, where the experts'
           results are weighted and summed, `head` from tokens to tokens.
  route    b200_op_route: the router in front of them: the chosen experts, their weights, and the requests sorted by expert.
  heads    b200_op_qk_norm_rotate: norms of queries and keys for each head with the position rotation in the same pass.
"""
import ctypes
import math

import numpy as np
import torch

own = False

DTYPE = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
PREC = {"fp32": 0, "fp16": 1, "bf16": 2}
ACTS = {"mish": 1, "none": 3, "swish": 7, "relu2": 8}


def listed():
    return [
        # One position at the root of a search, an encoder product of the BT4-class network: 64 rows; latency.
        dict(name="int8_root", op="int8", type="fp16", rows=64, n=1024, k=1024, act="none", res=False, f32=False),
        # The batch of the headline throughput: the FFN's second product with its residual.
        dict(name="int8_body_1024", op="int8", type="bf16", rows=1024 * 64, n=1024, k=1536, act="none", res=True, f32=False),
        # The classical policy head (32 planes x 64 squares -> 1858 logits in fp32) of a few positions, odd numbers of rows and columns.
        dict(name="int8_policy_37", op="int8", type="fp16", rows=37, n=1858, k=2048, act="none", res=False, f32=True),
        # A search's minibatch of 24 positions; each position picks its expert (opening, middlegame, ...), three have none.
        dict(name="experts_search_24", op="experts", type="fp16", int8=False, side="up", requests=24, group=64, experts=8, top_k=1,
             n=1536, k=1024, act="relu2", res=False, f32=False, drop=True),
        # Token-wise experts over a throughput batch of 256 positions, two experts per token: into the hidden layer, and back.
        dict(name="experts_up_16384", op="experts", type="bf16", int8=False, side="up", requests=16384, group=1, experts=16, top_k=2,
             n=1536, k=1024, act="mish", res=False, f32=False, drop=False),
        dict(name="experts_down_16384", op="experts", type="fp16", int8=False, side="down", requests=16384, group=1, experts=16, top_k=2,
             n=1024, k=1536, act="none", res=True, f32=False, drop=False),
        # The same in 8 bits at a ragged batch.
        dict(name="experts_int8_9000", op="experts", type="bf16", int8=True, side="up", requests=9000, group=1, experts=16, top_k=2,
             n=1536, k=1024, act="mish", res=False, f32=False, drop=False),
        # A policy head per expert, one row per position, ragged, logits in fp32.
        dict(name="experts_policy_333", op="experts", type="bf16", int8=False, side="head", requests=333, group=1, experts=12, top_k=1,
             n=1858, k=1024, act="none", res=False, f32=True, drop=True),
        # The router of a search's minibatch, and of the headline batch with many experts.
        dict(name="route_1536", op="route", type="fp32", rows=1536, experts=16, top_k=2, renormalise=True),
        dict(name="route_65536", op="route", type="bf16", rows=65536, experts=64, top_k=4, renormalise=False),
        # Queries and keys of one position; of the headline batch, packed beside the values.
        dict(name="heads_root", op="heads", type="fp16", rows=64, q_heads=32, k_heads=32, depth=32, rotate=32, interleaved=False, packed=False),
        dict(name="heads_body_1024", op="heads", type="bf16", rows=1024 * 64, q_heads=24, k_heads=24, depth=32, rotate=32, interleaved=True, packed=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["int8", "int8", "experts", "experts", "experts", "route", "heads"])
    t = rng.choice(["fp16", "bf16"])
    if op == "int8":
        c = dict(op=op, type=t, n=rng.choice([32, 128, 256, 512, 1000, 1024, 1536, 1858]), k=rng.choice([64, 256, 512, 624, 1024, 1536, 2048]),
                 act=rng.choice(["none", "mish", "swish", "relu2"]), res=rng.random() < 0.4, f32=rng.random() < 0.2)
        rows = 64 * _log(rng, 1, 1024) if rng.random() < 0.6 else _log(rng, 1, 4096)
        row_bytes = 2 * c["k"] + (4 if c["f32"] else 2) * c["n"] * (2 if c["res"] else 1)
        c["rows"] = max(1, min(rows, 65536 * 1536 * 1024 // (c["n"] * c["k"]), 460_000_000 // row_bytes))
        return c
    if op == "experts":
        c = dict(op=op, type=t, int8=rng.random() < 0.35, side=rng.choice(["up", "up", "down", "head"]),
                 n=rng.choice([128, 256, 512, 768, 1024, 1536, 1858]), k=rng.choice([128, 256, 512, 768, 1024, 1536]),
                 act=rng.choice(["none", "mish", "swish", "relu2"]), experts=_log(rng, 2, 64), drop=rng.random() < 0.3)
        c["group"] = rng.choice([1, 1, 64])
        c["top_k"] = 1 if c["group"] > 1 or c["side"] == "head" else min(c["experts"], rng.choice([1, 2, 2, 4]))
        c["res"] = c["side"] != "up" and rng.random() < 0.5
        c["f32"] = c["side"] == "head" and rng.random() < 0.4
        c["requests"] = max(1, min(_log(rng, 1, 20000) if c["group"] == 1 else _log(rng, 1, 400),
                                   32768 * 1536 * 1024 // (c["n"] * c["k"] * c["group"] * c["top_k"])))
        return c
    if op == "route":
        c = dict(op=op, type=rng.choice(["fp32", "fp16", "bf16"]), rows=_log(rng, 1, 65536), experts=_log(rng, 2, 256), renormalise=rng.random() < 0.5)
        c["top_k"] = min(c["experts"], rng.choice([1, 2, 2, 4, 8]))
        return c
    depth = rng.choice([16, 32, 32, 64, 96, 128])
    heads = rng.choice([4, 8, 16, 24, 32])
    c = dict(op=op, type=rng.choice(["fp16", "bf16", "fp32"]), q_heads=heads, k_heads=heads // rng.choice([1, 1, 2, 4]), depth=depth,
             rotate=rng.choice([0, depth // 2, depth, depth]), interleaved=rng.random() < 0.5, packed=rng.random() < 0.5)
    c["rows"] = max(1, min(64 * _log(rng, 1, 1024), 65536 * 48 * 32 // ((c["q_heads"] + c["k_heads"]) * depth * (2 if c["type"] == "fp32" else 1))) - rng.choice([0, 0, 1, 13]))
    return c


def _inputs(case, seed):
    """The case's inputs from its seed: activations of order one with a few large channels, weights of fan-in scale, routers with
    popular and unpopular experts."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    def whole(*shape):  # 8-bit values of normal spread
        return rnd(*shape).mul_(36).round_().clamp_(-127, 127).to(torch.int8)

    t = DTYPE[case["type"]]
    if case["op"] == "int8":
        m, n, k = case["rows"], case["n"], case["k"]
        d = dict(x=(rnd(m, k) * (1 + 7 * (rand(k) < 0.01))).to(t), w=whole(n, k), w_scales=(0.5 + rand(n)) * k ** -0.5 / 36, bias=rnd(n) * 0.1)
        if case["res"]:
            d["res"] = rnd(m, n).to(torch.float32 if case["f32"] else t)
        return d
    if case["op"] == "experts":
        e, k, n, top, requests, group = (case[x] for x in ("experts", "k", "n", "top_k", "requests", "group"))
        logits = rnd(requests, e) + rnd(e)
        ids = logits.topk(top, dim=1).indices.int()
        if case["drop"]:
            ids = torch.where(rand(requests, 1) < 0.125, -1, ids).int()
        flat = ids.reshape(-1)
        key = torch.where(flat < 0, e, flat).long()
        rows = requests * group * (top if case["side"] == "down" else 1)
        d = dict(ids=ids, order=torch.argsort(key, stable=True).int(),
                 offsets=torch.cat([key.new_zeros(1), torch.bincount(key, minlength=e + 1)[:e].cumsum(0)]).int(), bias=rnd(e, n) * 0.1)
        if case["int8"]:
            d.update(x=whole(rows, k), x_scales=(0.5 + rand(rows)) / 36, w=whole(e, n, k), w_scales=(0.5 + rand(e, n)) * k ** -0.5 / 36)
        else:
            d.update(x=rnd(rows, k).to(t), w=torch.stack([(rnd(n, k) * k ** -0.5).to(t) for _ in range(e)]))
        if case["side"] == "down":
            d["weights"] = torch.softmax(rnd(requests, top), dim=1)
        if case["res"]:
            d["res"] = rnd(requests * group, n).to(torch.float32 if case["f32"] else t)
        return d
    if case["op"] == "route":
        return dict(logits=(rnd(case["rows"], case["experts"]) * 1.5 + rnd(case["experts"])).to(t))
    rows, hq, hk, depth, rot = (case[x] for x in ("rows", "q_heads", "k_heads", "depth", "rotate"))
    d = dict(gamma_q=1 + 0.2 * rnd(depth), gamma_k=1 + 0.2 * rnd(depth))
    if case["packed"]:  # queries, keys and values side by side, as one product writes them
        qkv = rnd(rows, (hq + 2 * hk) * depth).to(t)
        d.update(q=qkv[:, :hq * depth], k=qkv[:, hq * depth:(hq + hk) * depth])
    else:
        d.update(q=rnd(rows, hq * depth).to(t), k=rnd(rows, hk * depth).to(t))
    if rot:  # a table for the 64 squares: half of the pairs turn with the file, half with the rank
        square = torch.arange(64, device="cuda", dtype=torch.float64)
        pair = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
        angle = torch.where(pair % 2 == 0, square[:, None] % 8, square[:, None] // 8) * 100.0 ** (-pair / (rot // 2))
        d["table"] = torch.stack([angle.cos(), angle.sin()], dim=2).float().contiguous()
    return d


def prepare(case, seed):
    s = dict(case=case, **_inputs(case, seed))
    torch.cuda.synchronize()
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------
def _activate(v, act):
    if act == "mish":
        return v * torch.tanh(torch.log1p(torch.exp(-v.abs())) + v.clamp(min=0))
    if act == "swish":
        return v / (1 + torch.exp(-v))
    return v.clamp(min=0) ** 2 if act == "relu2" else v


def _int8_plain(s):
    c = s["case"]
    x = s["x"].float()
    scale = x.abs().amax(dim=1, keepdim=True) / 127
    q = torch.where(scale > 0, torch.round(x.double() / scale.double()), 0.0).clamp(-127, 127).float()  # quotients next to a half need 64 bits
    y = _activate((q @ s["w"].float().T) * (scale * s["w_scales"]) + s["bias"], c["act"])
    if c["res"]:
        y = y + s["res"].float()
    return y if c["f32"] else y.to(s["x"].dtype)


def _experts_plain(s):
    c = s["case"]
    group, top, out_type = c["group"], c["top_k"], torch.float32 if c["f32"] else DTYPE[c["type"]]
    tokens = c["requests"] * group
    inside = torch.arange(group, device="cuda")
    y = torch.zeros(tokens * top, c["n"], device="cuda")  # by slot ("up") or by request and choice
    at = s["offsets"].tolist()
    for e in range(c["experts"]):
        if at[e] == at[e + 1]:
            continue
        chosen = s["order"][at[e]:at[e + 1]].long()
        rows = ((chosen // top)[:, None] * group + inside).view(-1)
        slots = slice(at[e] * group, at[e + 1] * group)
        x = s["x"][slots] if c["side"] == "down" else s["x"][rows]
        v = x.float() @ s["w"][e].float().T
        if c["int8"]:
            v = v * ((s["x_scales"][slots] if c["side"] == "down" else s["x_scales"][rows])[:, None] * s["w_scales"][e])
        v = _activate(v + s["bias"][e], c["act"])
        if c["side"] == "up":
            y[slots] = v
        else:
            if "weights" in s:
                v = v * s["weights"].view(-1)[chosen].repeat_interleave(group)[:, None]
            y[(chosen[:, None] * group + inside).view(-1)] = v
    if c["side"] != "up":
        y = y.view(c["requests"], top, group, c["n"]).sum(1).view(tokens, c["n"])
        if c["res"]:
            y = torch.where((s["ids"] >= 0).any(dim=1).repeat_interleave(group)[:, None], y + s["res"].float(), 0.0)
    return y.to(out_type)


def _route_plain(s):
    c = s["case"]
    l = s["logits"].float()
    e, top = c["experts"], c["top_k"]
    first = torch.sort(l, dim=1, descending=True, stable=True)
    chosen, ids = first.values[:, :top], first.indices[:, :top].int()
    w = torch.exp(chosen - chosen[:, :1])
    total = w if c["renormalise"] else torch.exp(l - chosen[:, :1])
    flat = ids.reshape(-1).long()
    offsets = torch.cat([flat.new_zeros(1), (flat[None, :] == torch.arange(e, device="cuda")[:, None]).sum(1).cumsum(0)]).int()
    return ids, w / total.sum(dim=1, keepdim=True), torch.sort(flat, stable=True).indices.int(), offsets


def _heads_plain(s):
    c = s["case"]
    out = []
    for x, heads, gamma in ((s["q"], c["q_heads"], s["gamma_q"]), (s["k"], c["k_heads"], s["gamma_k"])):
        v = x.float().reshape(c["rows"], heads, c["depth"])
        v = v / torch.sqrt((v * v).mean(dim=2, keepdim=True) + 1e-6) * gamma
        if c["rotate"]:
            turn = s["table"][torch.arange(c["rows"], device="cuda") % 64][:, None]
            cos, sin = turn[..., 0], turn[..., 1]
            r = c["rotate"]
            a, b = (v[..., 0:r:2], v[..., 1:r:2]) if c["interleaved"] else (v[..., :r // 2], v[..., r // 2:r])
            a, b = a * cos - b * sin, a * sin + b * cos
            turned = torch.stack([a, b], dim=3).reshape(c["rows"], heads, r) if c["interleaved"] else torch.cat([a, b], dim=2)
            v = torch.cat([turned, v[..., r:]], dim=2)
        out.append(v.reshape(c["rows"], heads * c["depth"]).to(x.dtype))
    return tuple(out)


# ---- the framework's operators ----------------------------------------------------------------------------------
def _workspace(lib, size_of, d):
    from lc0_b200 import _lib
    need = ctypes.c_size_t()
    _lib.check(size_of(ctypes.byref(d), ctypes.byref(need)))
    work = torch.empty(max(need.value, 1), dtype=torch.uint8, device="cuda")
    d.workspace, d.workspace_bytes = work.data_ptr(), need.value
    return work


def _own(s):
    """Descriptions of the calls, outputs and workspaces: made at a state's first pass and kept, as a program does."""
    from lc0_b200 import _lib
    lib, c = _lib.load(), s["case"]
    prec = PREC[c["type"]]

    def p(name):
        return s[name].data_ptr() if name in s else None

    def empty(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    if c["op"] == "int8":
        m, n, k = c["rows"], c["n"], c["k"]
        q, scales, out = empty(m, k, dtype=torch.int8), empty(m), empty(m, n, dtype=torch.float32 if c["f32"] else DTYPE[c["type"]])
        d = _lib.GemmInt8Desc(X=q.data_ptr(), x_scales=scales.data_ptr(), W=p("w"), w_scales=p("w_scales"), bias=p("bias"), C=out.data_ptr(), M=m, N=n, K=k,
                              activation=ACTS[c["act"]], precision=0 if c["f32"] else prec, alpha=1.0, res=p("res"), status=status.data_ptr())
        calls = [(lib.b200_op_quantize_rows, (p("x"), 0, m, k, prec, q.data_ptr(), 0, scales.data_ptr())), (lib.b200_op_gemm_int8, (ctypes.byref(d),))]
        return _lib.check, calls, out, (q, scales, d, status)
    if c["op"] == "experts":
        tokens = c["requests"] * c["group"]
        by_slot = c["side"] == "up"
        out = torch.zeros(tokens * (c["top_k"] if by_slot else 1), c["n"], dtype=torch.float32 if c["f32"] else DTYPE[c["type"]], device="cuda")
        d = _lib.ExpertsDesc(X=p("x"), W=p("w"), bias=p("bias"), C=out.data_ptr(), M=tokens, N=c["n"], K=c["k"], activation=ACTS[c["act"]], precision=prec,
                             out_f32=int(c["f32"]), int8=int(c["int8"]), x_scales=p("x_scales"), w_scales=p("w_scales"), n_experts=c["experts"],
                             top_k=c["top_k"], group=c["group"], ids=p("ids"), order=p("order"), offsets=p("offsets"), x_by_slot=int(c["side"] == "down"),
                             c_by_slot=int(by_slot), weights=p("weights"), res=p("res"), status=status.data_ptr())
        work = _workspace(lib, lib.b200_op_gemm_experts_workspace, d)
        return _lib.check, [(lib.b200_op_gemm_experts, (ctypes.byref(d),))], out, (d, work, status)
    if c["op"] == "route":
        rows, top = c["rows"], c["top_k"]
        out = (empty(rows, top, dtype=torch.int32), empty(rows, top), empty(rows * top, dtype=torch.int32), empty(c["experts"] + 1, dtype=torch.int32))
        d = _lib.RouteDesc(logits=p("logits"), rows=rows, n_experts=c["experts"], top_k=top, precision=prec, renormalise=int(c["renormalise"]),
                           ids=out[0].data_ptr(), weights=out[1].data_ptr(), order=out[2].data_ptr(), offsets=out[3].data_ptr())
        work = _workspace(lib, lib.b200_op_route_workspace, d)
        return _lib.check, [(lib.b200_op_route, (ctypes.byref(d),))], out, (d, work)
    out = tuple(empty(c["rows"], c[h] * c["depth"], dtype=DTYPE[c["type"]]) for h in ("q_heads", "k_heads"))
    d = _lib.QkNormDesc(q=p("q"), k=p("k"), ldq=s["q"].stride(0), ldk=s["k"].stride(0), q_out=out[0].data_ptr(), k_out=out[1].data_ptr(), rows=c["rows"],
                        q_heads=c["q_heads"], k_heads=c["k_heads"], depth=c["depth"], precision=prec, norm=1, eps=1e-6, gamma_q=p("gamma_q"),
                        gamma_k=p("gamma_k"), rotate=c["rotate"], interleaved=int(c["interleaved"]), table=p("table"), n_positions=64 if c["rotate"] else 0)
    return _lib.check, [(lib.b200_op_qk_norm_rotate, (ctypes.byref(d),))], out, (d,)


def run(s):
    if own:
        if "calls" not in s:
            s["calls"] = _own(s)
        check, calls, out, _ = s["calls"]
        stream = torch.cuda.current_stream().cuda_stream
        for op, args in calls:
            check(op(*args, stream))
        return out
    return {"int8": _int8_plain, "experts": _experts_plain, "route": _route_plain, "heads": _heads_plain}[s["case"]["op"]](s)


# ---- definitions in 64 bits -------------------------------------------------------------------------------------
def _activate_exact(v, act):
    if act == "mish":
        return v * torch.tanh(torch.logaddexp(v, torch.zeros_like(v)))
    if act == "swish":
        return v * torch.sigmoid(v)
    return torch.relu(v).square() if act == "relu2" else v


def _int8_exact(c, d):
    out = torch.empty(c["rows"], c["n"], dtype=torch.float64, device="cuda")
    w = d["w"].double() * d["w_scales"].double()[:, None]
    for i in range(0, c["rows"], 8192):
        x = d["x"][i:i + 8192].double()
        scale = (x.abs().max(dim=1).values.float() / 127).double()  # the scale is a number of 32 bits
        q = torch.round(x / torch.where(scale > 0, scale, 1.0)[:, None]).clamp(-127, 127)
        v = _activate_exact((q * scale[:, None]) @ w.T + d["bias"].double(), c["act"])
        out[i:i + 8192] = v + d["res"][i:i + 8192].double() if c["res"] else v
    return out


def _experts_exact(c, d):
    group, top = c["group"], c["top_k"]
    ids = d["ids"].repeat_interleave(group, dim=0)  # [tokens][top_k]
    out = torch.zeros(ids.shape[0] * (top if c["side"] == "up" else 1), c["n"], dtype=torch.float64, device="cuda")
    slot = torch.empty(c["requests"] * top, dtype=torch.long, device="cuda")
    slot[d["order"].long()] = torch.arange(c["requests"] * top, device="cuda")
    if c["res"]:
        out[(ids >= 0).any(dim=1)] = d["res"][(ids >= 0).any(dim=1)].double()
    for e in range(c["experts"]):
        for j in range(top):
            token = (ids[:, j] == e).nonzero()[:, 0]
            if token.numel() == 0:
                continue
            by_slot = slot[(token // group) * top + j] * group + token % group
            source = by_slot if c["side"] == "down" else token
            x, w = d["x"][source].double(), d["w"][e].double()
            if c["int8"]:
                x, w = x * d["x_scales"][source].double()[:, None], w * d["w_scales"][e].double()[:, None]
            v = _activate_exact(x @ w.T + d["bias"][e].double(), c["act"])
            if "weights" in d:
                v = v * d["weights"][token // group, j].double()[:, None]
            if c["side"] == "up":
                out[by_slot] = v
            else:
                out[token] += v
    return out


def _route_exact(c, d):
    l = d["logits"].double().cpu().numpy()
    e, top = c["experts"], c["top_k"]
    ids = np.argsort(-l, axis=1, kind="stable")[:, :top]
    w = np.exp(l - l.max(axis=1, keepdims=True))
    chosen = np.take_along_axis(w, ids, axis=1)
    weights = chosen / (chosen if c["renormalise"] else w).sum(axis=1, keepdims=True)
    flat = ids.reshape(-1)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=e))])
    return (torch.from_numpy(ids.astype(np.int32)), torch.from_numpy(weights), torch.from_numpy(np.argsort(flat, kind="stable").astype(np.int32)),
            torch.from_numpy(offsets.astype(np.int32)))


def _heads_exact(c, d):
    out = []
    for name, heads in (("q", c["q_heads"]), ("k", c["k_heads"])):
        v = d[name].double().reshape(c["rows"], heads, c["depth"])
        v = v * torch.rsqrt(v.square().mean(dim=2, keepdim=True) + float(np.float32(1e-6))) * d["gamma_" + name].double()
        if c["rotate"]:
            half = c["rotate"] // 2
            pair = torch.arange(half, device="cuda")
            ia, ib = (2 * pair, 2 * pair + 1) if c["interleaved"] else (pair, pair + half)
            table = d["table"].double().repeat((c["rows"] + 63) // 64, 1, 1)[:c["rows"], None]
            z = torch.complex(v[..., ia], v[..., ib]) * torch.complex(table[..., 0], table[..., 1])
            v[..., ia], v[..., ib] = z.real, z.imag
        out.append(v.reshape(c["rows"], heads * c["depth"]))
    return tuple(out)


def exact(case, seed):
    return {"int8": _int8_exact, "experts": _experts_exact, "route": _route_exact, "heads": _heads_exact}[case["op"]](case, _inputs(case, seed))


# ---- work -------------------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] == "int8":
        m, n, k = case["rows"], case["n"], case["k"]
        out = 4 if case["f32"] else size
        return {"bytes": m * k * size + n * k + 8 * n + m * n * out * (2 if case["res"] else 1), "flops": 2 * m * n * k + 4 * m * k}
    if case["op"] == "experts":
        n, k, e, top = (case[x] for x in ("n", "k", "experts", "top_k"))
        requests = case["requests"] * (7 / 8 if case["drop"] else 1)
        rows = requests * case["group"]
        slots = rows * top
        unit, out = 1 if case["int8"] else size, 4 if case["f32"] else size
        used = e * (1 - (1 - 1 / e) ** (requests * top))  # expected number of experts in use, were all as popular
        moved = (slots if case["side"] == "down" else rows) * (k * unit + 4 * case["int8"]) + used * n * (k * unit + 4 + 4 * case["int8"])
        moved += (slots if case["side"] == "up" else rows * (2 if case["res"] else 1)) * n * out + 4 * requests * top
        return {"bytes": moved + (4 * requests * top if case["side"] == "down" else 0), "flops": 2 * slots * n * k}
    if case["op"] == "route":
        return {"bytes": case["rows"] * (case["experts"] * size + 12 * case["top_k"]) + 4 * case["experts"], "flops": case["rows"] * case["experts"] * 8}
    entries = case["rows"] * (case["q_heads"] + case["k_heads"]) * case["depth"]
    return {"bytes": 2 * size * entries + 64 * 4 * case["rotate"] + 8 * case["depth"], "flops": 8 * entries}
