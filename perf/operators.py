"""Cases of two operators of a served mixture-of-experts layer: the choice of experts from a token's logits
(lowoha.moe_router_grouped) and the low-rank adapters of many requests beside a shared projection (lowoha.lora_direct).

`run` computes a case with elementary torch operations, or, with `own` set, with the framework's calls.  `exact` gives
the same outputs from the operators' definitions in 64 bits."""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _router(name, T, E, topk, dt, scoring, bias, n_group=1, topk_group=1, top2=False, renormalize=True, scale=1.0, pad=0):
    return {"name": name, "op": "router", "T": T, "E": E, "topk": topk, "dt": dt, "scoring": scoring, "bias": bias,
            "n_group": n_group, "topk_group": topk_group, "top2": top2, "renormalize": renormalize, "scale": scale, "pad": pad}


def _lora(name, T, K, N0, N1, N2, rank, slots, dt, dst, mixed=True, pad=0):
    return {"name": name, "op": "lora", "T": T, "K": K, "N0": N0, "N1": N1, "N2": N2, "rank": rank, "slots": slots, "dt": dt,
            "dst": dst, "mixed": mixed, "pad": pad}


def listed():
    return [
        # one generated token of one request: sigmoid scores, a balancing bias, 4 of 8 groups, 8 of 256 experts
        _router("router_1x256", 1, 256, 8, "f32", "sigmoid", True, 8, 4, True, True, 2.5),
        # a decode batch of a model with few experts; the gate projection leaves bf16 logits
        _router("router_64x64_bf16", 64, 64, 6, "bf16", "softmax", False),
        # a chunk of prompts on an odd number of experts in groups ranked by their best expert, rows inside a wider buffer
        _router("router_777x60_f16", 777, 60, 5, "f16", "softmax", True, 5, 2, False, False, 1.0, 20),
        # a long prefill of the first case's model
        _router("router_8192x256", 8192, 256, 8, "f32", "sigmoid", True, 8, 4, True, True, 2.5),
        # a whole batch of prompts, many experts without groups
        _router("router_32768x512", 32768, 512, 10, "f32", "softmax", True),
        # one generated token of one request beside an output projection
        _lora("lora_1x4096x4096_r16", 1, 4096, 4096, 0, 0, 16, 4, "bf16", "bf16"),
        # a decode batch, almost every row another adapter, beside a fused query / key / value projection
        _lora("lora_48_qkv_r64", 48, 4096, 4096, 1024, 1024, 64, 64, "bf16", "bf16"),
        # a decode batch on a down projection (long rows), few adapters
        _lora("lora_128x14336x4096_r16", 128, 14336, 4096, 0, 0, 16, 6, "bf16", "bf16"),
        # a chunk of prompts: odd sizes, an odd rank, f16, rows inside wider buffers
        _lora("lora_301x1001x2731_r12_f16", 301, 1001, 2731, 0, 0, 12, 9, "f16", "f16", True, 7),
        # prompts of requests with adapters on the gate projection: f32 logits, few columns
        _lora("lora_2048_gate_r8", 2048, 4096, 256, 0, 0, 8, 16, "bf16", "f32"),
        # prefill of a fused gate / up projection
        _lora("lora_2048_gate_up_r32", 2048, 4096, 14336, 14336, 0, 32, 4, "bf16", "bf16"),
        # a whole batch of prompts on a down projection with high-rank adapters
        _lora("lora_8192x14336x4096_r128", 8192, 14336, 4096, 0, 0, 128, 8, "bf16", "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _unnamed(case):
    del case["name"]
    return case


def draw(rng):
    if rng.random() < 0.4:
        dt, scoring = rng.choice(["f32", "bf16", "f16"]), rng.choice(["softmax", "sigmoid"])
        n_group = rng.choice([1, 1, 2, 3, 4, 8])
        per = max(2, _log(rng, 4, 512) // n_group)
        E = n_group * per
        topk_group = rng.randint(1, n_group)
        topk = min(rng.randint(1, 16), topk_group * per)
        return _unnamed(_router("", _log(rng, 1, 16384), E, topk, dt, scoring, rng.random() < 0.6, n_group, topk_group,
                       n_group > 1 and rng.random() < 0.5, rng.random() < 0.5, rng.choice([1.0, 2.5]), rng.choice([0, 0, 13])))
    dt = rng.choice(["bf16", "bf16", "f16"])
    dst = rng.choice([dt, dt, "f32"])
    odd = rng.random() < 0.3
    T, K, N0 = _log(rng, 1, 4096), _log(rng, 128, 14336), _log(rng, 64, 14336)
    N1, N2 = (0, 0) if rng.random() < 0.6 else (_log(rng, 64, 4096), rng.choice([0, 1024]))
    if not odd:
        K, N0, N1 = K // 8 * 8, N0 // 8 * 8, N1 // 8 * 8
    rank = rng.choice([1, 4, 8, 12, 16, 16, 24, 32, 64, 128])
    # (no more than the largest listed case: the plain form's products go over all slots)
    most = 8192 * 8 * 128 * (14336 + 4096) // (T * rank * ((1 + (N1 > 0) + (N2 > 0)) * K + N0 + N1 + N2))
    slots = _log(rng, 1, max(1, min(64, most)))
    return _unnamed(_lora("", T, K, N0, N1, N2, rank, slots, dt, dst, rng.random() < 0.7, rng.choice([0, 0, 8, 5])))


def _rows(g, T, C, pad, dt, std=1.0):
    """[T, C] rows of a buffer that is `pad` elements wider."""
    return (torch.randn(T, C + pad, generator=g, device=DEV) * std).to(TYPES[dt])[:, :C]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    c, T = case, case["T"]
    if c["op"] == "router":
        E = c["E"]
        # a gate projection's logits: some experts are liked more than others
        x = torch.randn(T, E + c["pad"], generator=g, device=DEV) * 1.5 + torch.randn(E + c["pad"], generator=g, device=DEV) * 0.7
        bias = torch.randn(E, generator=g, device=DEV) * 0.05 if c["bias"] else None
        return {"case": c, "logits": x.to(TYPES[c["dt"]])[:, :E], "bias": bias}
    K, R, S = c["K"], c["rank"], c["slots"]
    N = [n for n in (c["N0"], c["N1"], c["N2"]) if n]
    x = _rows(g, T, K, c["pad"], c["dt"])
    a = (torch.randn(S, len(N) * R, K, generator=g, device=DEV) / math.sqrt(K)).to(TYPES[c["dt"]])
    b = [(torch.randn(S, n, R, generator=g, device=DEV) * 0.1).to(TYPES[c["dt"]]) for n in N]
    ids = torch.randint(0, S, (T,), generator=g, device=DEV, dtype=torch.int32)
    if T > 8:   # one row in eight belongs to a request without an adapter
        ids = torch.where(torch.rand(T, generator=g, device=DEV) < 0.125, torch.full_like(ids, -1), ids)
    ranks = None
    if c["mixed"]:   # every other slot holds an adapter of half the rank (the slot's other rows are an earlier adapter's)
        ranks = torch.tensor([R if s % 2 == 0 else max(1, R // 2) for s in range(S)], dtype=torch.int32, device=DEV)
    scales = torch.rand(S, generator=g, device=DEV) + 0.5
    base = _rows(g, T, sum(N), c["pad"], c["dst"])
    out = torch.empty(T, sum(N), dtype=TYPES[c["dst"]], device=DEV)
    return {"case": c, "x": x, "a": a, "b": b, "ids": ids, "ranks": ranks, "scales": scales, "base": base, "out": out}


def _router_plain(s):
    c = s["case"]
    T, E, G = c["T"], c["E"], c["n_group"]
    x = s["logits"].double()   # (two experts' values may be nearer than 32 bits can tell)
    if c["scoring"] == "sigmoid":
        p = 1.0 / (1.0 + torch.exp(-x))
    else:
        e = torch.exp(x - x.amax(1, keepdim=True))
        p = e / e.sum(1, keepdim=True)
    v = p + s["bias"].double() if s["bias"] is not None else p
    if G > 1:
        by_group = v.view(T, G, E // G)
        best = by_group.sort(2, descending=True).values[:, :, :2].sum(2) if c["top2"] else by_group.amax(2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["topk_group"]]
        live = torch.zeros(T, G, dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        v = torch.where(live[:, :, None], by_group, torch.full_like(by_group, -math.inf)).view(T, E)
    ids = torch.sort(v, dim=1, descending=True, stable=True).indices[:, :c["topk"]]
    w = torch.gather(p, 1, ids)
    if c["renormalize"]:
        w = w / w.sum(1, keepdim=True)
    return [ids.int(), (w * c["scale"]).float()]


def _lora_plain(s):
    c = s["case"]
    T, K, R, S = c["T"], c["K"], c["rank"], c["slots"]
    ids = s["ids"].long()
    # the products with every slot's adapter; those of other slots than the row's own are dropped
    mine = torch.arange(S, device=ids.device)[None, :] == ids[:, None]
    live = mine[:, :, None].expand(T, S, R)
    if s["ranks"] is not None:
        live = live & (torch.arange(R, device=ids.device)[None, :] < s["ranks"][:, None])[None]
    h = (s["x"].float() @ s["a"].float().view(-1, K).t()).view(T, S, -1, R)
    h = torch.where(live[:, :, None, :], h * s["scales"][None, :, None, None], torch.zeros((), device=h.device))
    delta = torch.cat([h[:, :, i].reshape(T, S * R) @ b.float().transpose(1, 2).reshape(S * R, -1) for i, b in enumerate(s["b"])], 1)
    return (s["base"].float() + delta).to(TYPES[c["dst"]])


def run(state):
    if not own:
        return _router_plain(state) if state["case"]["op"] == "router" else _lora_plain(state)
    from zendnn_amd import capi, lowoha
    c = state["case"]
    if "call" not in state:   # the argument block that a serving loop keeps: addresses and sizes, no values
        if c["op"] == "router":
            state["call"], *state["got"] = lowoha.prepared_moe_router_grouped(
                state["logits"], c["topk"], scoring=capi.SCORE_SIGMOID if c["scoring"] == "sigmoid" else capi.SCORE_SOFTMAX,
                bias=state["bias"], n_group=c["n_group"], topk_group=c["topk_group"],
                group_score=capi.GROUP_TOP2_SUM if c["top2"] else capi.GROUP_MAX, renormalize=c["renormalize"], scale=c["scale"])
        else:
            state["call"] = lowoha.prepared_lora(state["x"], state["ids"], state["a"], state["b"], state["out"], base=state["base"],
                                                 ranks=state["ranks"], scales=state["scales"])
            state["got"] = state["out"]
    st = state["call"]()
    if st != capi.SUCCESS:
        raise RuntimeError(lowoha.last_error())
    return state["got"]


def work(case):
    c, T = case, case["T"]
    if c["op"] == "router":
        return {"bytes": T * c["E"] * SIZE[c["dt"]] + (4 * c["E"] if c["bias"] else 0) + 8 * T * c["topk"], "flops": 4 * T * c["E"]}
    N, n_slices = c["N0"] + c["N1"] + c["N2"], 1 + (c["N1"] > 0) + (c["N2"] > 0)
    S, rows = c["slots"], T * (0.875 if T > 8 else 1.0)   # (rows that have an adapter, slots that some row uses: on average)
    used = S * (1.0 - (1.0 - 1.0 / S) ** rows)
    rank = c["rank"]
    if c["mixed"]:
        rank = sum(rank if s % 2 == 0 else max(1, rank // 2) for s in range(S)) / S
    data = T * c["K"] * SIZE[c["dt"]] + 2 * T * N * SIZE[c["dst"]] + 4 * T
    return {"bytes": int(data + used * rank * (n_slices * c["K"] + N) * SIZE[c["dt"]]), "flops": int(2 * rows * rank * (n_slices * c["K"] + N))}


def exact(case, seed):
    s = prepare(case, seed)
    c, T = case, case["T"]
    if c["op"] == "router":
        E, G, k = c["E"], c["n_group"], c["topk"]
        x = s["logits"].double()
        p = torch.sigmoid(x) if c["scoring"] == "sigmoid" else torch.softmax(x, 1)
        v = p.clone() if s["bias"] is None else p + s["bias"].double()
        row = torch.arange(T, device=x.device)
        if G > 1:
            u = v.clone().view(T, G, -1)
            best, at = u.max(2)
            if c["top2"]:
                best = best + u.scatter(2, at[:, :, None], -math.inf).amax(2)
            allowed = torch.zeros(T, G, dtype=torch.bool, device=x.device)
            for _ in range(c["topk_group"]):
                i = best.amax(1, keepdim=True).eq(best).byte().argmax(1)
                allowed[row, i] = True
                best[row, i] = -math.inf
            v[~allowed.repeat_interleave(E // G, 1)] = -math.inf
        ids = []
        for _ in range(k):   # the first of the largest values that are left
            i = v.amax(1, keepdim=True).eq(v).byte().argmax(1)
            v[row, i] = -math.inf
            ids.append(i)
        ids = torch.stack(ids, 1)
        w = p[row[:, None], ids]
        return [ids.int(), c["scale"] * (w / w.sum(1, keepdim=True) if c["renormalize"] else w)]
    y = s["base"].double()
    R = c["rank"]
    for a in range(c["slots"]):
        rows = (s["ids"] == a).nonzero()[:, 0]
        if not len(rows):
            continue
        r = int(s["ranks"][a]) if s["ranks"] is not None else R
        x, col = s["x"][rows].double(), 0
        for i, b in enumerate(s["b"]):
            n = b.shape[1]
            y[rows, col:col + n] += float(s["scales"][a]) * ((x @ s["a"][a, i * R:i * R + r].double().t()) @ b[a, :, :r].double().t())
            col += n
    return y
