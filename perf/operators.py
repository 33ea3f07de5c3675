"""Timed cases of the two selections a decoded token goes through: the router in front of a layer's experts and the
draw of the next token from the head's logits.

The router scores a token's experts (softmax or sigmoid of its logits), adds a balance bias to choose by, keeps the
best groups of experts where the model has groups, and returns the best experts with their weights; a shared expert
takes a slot of its own.  The draw applies temperature, top-k, top-p and min-p, alike for all rows or each row its own, and
takes the token at the given random number.  Sizes are those of the 2048-wide model of the benchmark (256 routed
experts, 8 a token; 151,936 tokens) and other, odd ones.

A case is a dict.  ``kind`` "route": ``tokens``, ``experts``, ``k``, ``dtype``, ``scoring`` ("softmax" / "sigmoid"),
``bias``, ``groups``, ``keep`` (groups that stay), ``group_score`` ("max" / "top2"), ``renormalise``, ``scale``,
``shared`` (the token's activation and a gate vector given).  ``kind`` "sample": ``rows``, ``vocab``, ``dtype``,
``temperature``, ``top_k``, ``top_p``, ``min_p``, ``per_row`` (each row its own settings instead), ``masked`` (the last columns
are padding, -inf).
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
HIDDEN, VOCAB = 2048, 151936


def _route(name, tokens, experts, k, dtype, scoring="softmax", bias=False, groups=1, keep=1, group_score="max",
           renormalise=True, scale=1.0, shared=False):
    case = dict(kind="route", tokens=tokens, experts=experts, k=k, dtype=dtype, scoring=scoring, bias=bias, groups=groups,
                keep=keep, group_score=group_score, renormalise=renormalise, scale=scale, shared=shared)
    return dict(case, name=name) if name else case


def _sample(name, rows, vocab, dtype, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, per_row=False, masked=False):
    case = dict(kind="sample", rows=rows, vocab=vocab, dtype=dtype, temperature=temperature, top_k=top_k, top_p=top_p,
                min_p=min_p, per_row=per_row, masked=masked)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one decoded token through a layer's router: latency
        _route("route_t1", 1, 256, 8, "fp32", "sigmoid", True, 8, 4, "top2", True, 2.5, True),
        # a batch of decoded tokens, few experts, weights as the softmax gives them
        _route("route_t64", 64, 64, 6, "bf16", renormalise=False),
        # a prompt of odd length, experts not a power of two, groups by their best expert
        _route("route_t333", 333, 160, 6, "fp32", groups=8, keep=3, renormalise=False, scale=16.0),
        # a prompt's chunk, the shared expert's gate computed from the activation
        _route("route_t4096", 4096, 256, 8, "fp16", "sigmoid", shared=True),
        # a batch of prompts: biased and grouped
        _route("route_t16384", 16384, 256, 8, "bf16", "sigmoid", True, 8, 4, "top2", True, 2.5),
        # a batch of prompts over many experts, no groups
        _route("route_t32768", 32768, 512, 10, "fp32", "sigmoid", True),
        # one chat's next token, the usual settings
        _sample("sample_b1", 1, VOCAB, "fp32", 0.7, 50, 0.9),
        # one chat's next token by top-p alone
        _sample("sample_b1_p", 1, VOCAB, "fp32", 1.0, 0, 0.95),
        # a few sequences over a small vocabulary, a wide top-k
        _sample("sample_b8_k", 8, 32000, "fp16", 0.8, 1000),
        # a server's batch: every request has settings of its own; odd vocabulary with padded columns
        _sample("sample_b37", 37, 50257, "bf16", per_row=True, masked=True),
        # rollouts: the plain distribution, a large batch
        _sample("sample_b256_t", 256, VOCAB, "fp32"),
        # a large batch by top-p and min-p
        _sample("sample_b256", 256, VOCAB, "bf16", 0.9, 0, 0.9, 0.01),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if rng.random() < 0.5:
        experts = rng.choice([rng.randint(8, 512), 8 * rng.randint(2, 64)])
        groups = rng.choice([1, rng.choice([g for g in range(1, 33) if experts % g == 0])])
        keep = rng.randint(1, groups)
        k = rng.randint(1, min(12, keep * (experts // groups)))
        tokens = _log_int(rng, 1, 32768)
        return _route(None, tokens, experts, k, dtype, rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, groups, keep,
                      rng.choice(["max", "top2"]), rng.random() < 0.6, rng.choice([1.0, 2.5]),
                      tokens <= 4096 and rng.random() < 0.3)
    rows, vocab = _log_int(rng, 1, 256), _log_int(rng, 1000, VOCAB)
    return _sample(None, rows, vocab, dtype, rng.choice([1.0, rng.uniform(0.3, 1.5)]),
                   rng.choice([0, 0, _log_int(rng, 1, 2000)]), rng.choice([1.0, rng.uniform(0.5, 0.99)]),
                   rng.choice([0.0, 0.0, rng.uniform(0.005, 0.2)]), rng.random() < 0.3, rng.random() < 0.3)


# ------------------------------------------------------------------ inputs
def _route_inputs(case, g):
    T, E = case["tokens"], case["experts"]
    inp = {"logits": (torch.randn(T, E, generator=g, device=DEV) * 1.7).to(TYPES[case["dtype"]])}
    scale = 0.05 if case["scoring"] == "sigmoid" else 0.3 / E
    inp["bias"] = torch.randn(E, generator=g, device=DEV) * scale if case["bias"] else None
    if case["shared"]:
        inp["h"] = torch.randn(T, HIDDEN, generator=g, device=DEV).to(TYPES[case["dtype"]])
        inp["gate"] = (torch.randn(HIDDEN, generator=g, device=DEV) * 0.02).to(torch.float16)
    return inp


def _sample_inputs(case, g):
    B, V = case["rows"], case["vocab"]
    # the logits of a language model: a power law over tokens whose steepness changes from row to row, with noise
    steep = torch.rand(B, 1, generator=g, device=DEV) * 1.6 + 1.0
    rank = torch.rand(B, V, generator=g, device=DEV) * V + 2.0
    logits = 16.0 - steep * rank.log() + torch.randn(B, V, generator=g, device=DEV) * 0.4
    if case["masked"]:
        logits[:, V - V // 40:] = -math.inf
    inp = {"logits": logits.to(TYPES[case["dtype"]]), "u": torch.rand(B, generator=g, device=DEV)}

    def rows_of(lo, hi, off, part):
        """lo to hi, `off` for the given part of the rows"""
        v = torch.rand(B, generator=g, device=DEV) * (hi - lo) + lo
        return torch.where(torch.rand(B, generator=g, device=DEV) < part, torch.full_like(v, off), v)

    if case["per_row"]:
        inp.update(temperature=rows_of(0.5, 1.3, 0.0, 0.15), top_k=rows_of(1.0, 300.0, 0.0, 0.4).to(torch.int32),
                   top_p=rows_of(0.6, 0.99, 1.0, 0.3), min_p=rows_of(0.01, 0.1, 0.0, 0.6))
    else:
        inp.update({key: case[key] for key in ("temperature", "top_k", "top_p", "min_p")})
    return inp


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 1013 + 29)
    return (_route_inputs if case["kind"] == "route" else _sample_inputs)(case, g)


def prepare(case, seed):
    return dict(case=case, inp=_inputs(case, seed))


# ------------------------------------------------------- the operators' plain forms
def _plain_route(case, inp):
    E, k, G = case["experts"], case["k"], case["groups"]
    x = inp["logits"].double()  # (64 bits: choices next to a border)
    if case["scoring"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-x))
    else:
        e = torch.exp(x - x.amax(-1, keepdim=True))
        score = e / e.sum(-1, keepdim=True)
    choice = score if inp["bias"] is None else score + inp["bias"].double()
    if G > 1:
        per = choice.view(-1, G, E // G)
        if case["group_score"] == "max":
            best = per.amax(-1)
        else:
            best = torch.sort(per, dim=-1, descending=True)[0][..., :2].sum(-1)
        order = torch.sort(best, dim=-1, descending=True, stable=True)[1][:, :case["keep"]]
        stays = torch.zeros_like(best, dtype=torch.bool).scatter(1, order, True)
        choice = torch.where(stays.repeat_interleave(E // G, dim=1), choice, -math.inf)
    ids = torch.sort(choice, dim=-1, descending=True, stable=True)[1][:, :k]
    w = score.gather(1, ids)
    if case["renormalise"]:
        w = w / w.sum(-1, keepdim=True)
    w = (w * case["scale"]).float()
    ids = ids.to(torch.int32)
    if case["shared"]:
        dot = (inp["h"].float() * inp["gate"].float()).sum(-1, keepdim=True)
        ids = torch.cat([ids, torch.full_like(ids[:, :1], E)], dim=1)
        w = torch.cat([w, 1.0 / (1.0 + torch.exp(-dot))], dim=1)
    return ids, w


def _plain_sample(case, inp):
    logits, u = inp["logits"].float(), inp["u"]
    B, V = logits.shape

    def column(v, dtype):
        if not torch.is_tensor(v):  # (settings are held in 32 bits)
            v = torch.full((B,), v, dtype=torch.float32 if dtype.is_floating_point else dtype, device=DEV)
        return v.to(dtype).view(B, 1)

    t, p, m = (column(inp[key], torch.float64) for key in ("temperature", "top_p", "min_p"))
    k = column(inp["top_k"], torch.int64)
    k = torch.where(t <= 0, torch.ones_like(k), torch.where(k <= 0, torch.full_like(k, V), k))
    t = torch.where(t <= 0, torch.ones_like(t), t)
    best, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    w = torch.exp((best - best[:, :1]).double() / t)  # (64 bits: long sums, draws next to a border)
    w = torch.where(torch.arange(V, device=DEV) < k, w, 0.0)
    before = torch.cumsum(w, dim=-1) - w
    keep = (before < p * w.sum(-1, keepdim=True)) | (p >= 1.0)
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter(1, order, torch.where(keep & (w >= m), w, 0.0))
    run = torch.cumsum(kept, dim=-1)
    total = run[:, -1:]
    token = (run <= u.double().view(B, 1) * total).sum(-1, keepdim=True).clamp(max=V - 1)
    return token.view(B), torch.log(kept.gather(1, token) / total).float().view(B)


def _own_route(case, inp):
    from compressai_amd import kernels as K

    shared = dict(h=inp["h"], shared_gate=inp["gate"], shared_id=case["experts"]) if case["shared"] else {}
    return K.vq_router_select(inp["logits"], case["k"], scoring=case["scoring"], bias=inp["bias"], n_groups=case["groups"],
                              topk_groups=case["keep"], group_score=case["group_score"], renormalise=case["renormalise"],
                              scale=case["scale"], **shared)


def _own_sample(case, inp):
    from compressai_amd import kernels as K

    return K.vq_sample(inp["logits"], inp["u"], temperature=inp["temperature"], top_k=inp["top_k"], top_p=inp["top_p"],
                       min_p=inp["min_p"])


def run(state):
    case, inp = state["case"], state["inp"]
    if case["kind"] == "route":
        return (_own_route if own else _plain_route)(case, inp)
    return (_own_sample if own else _plain_sample)(case, inp)


# ------------------------------------------------- what a pass cannot do without
def work(case):
    size = BYTES[case["dtype"]]
    if case["kind"] == "route":
        T, E, slots = case["tokens"], case["experts"], case["k"] + case["shared"]
        moved = T * E * size + T * slots * 8 + case["bias"] * E * 4
        if case["shared"]:
            moved += T * HIDDEN * size + HIDDEN * 2
        # score and choice of every expert; the gate's product
        return {"bytes": moved, "flops": T * E * 4 + case["shared"] * T * HIDDEN * 2}
    B, V = case["rows"], case["vocab"]
    # difference, scaling, exponential and sum of every entry
    return {"bytes": B * V * size + B * (4 + 12) + case["per_row"] * B * 16, "flops": B * V * 4}


# --------------------------------------------- from the definitions, in 64 bits
def _exact_route(case, inp):
    x = inp["logits"].float().cpu().numpy().astype(np.float64)
    T, E = x.shape
    k, G, size = case["k"], case["groups"], E // case["groups"]
    if case["scoring"] == "sigmoid":
        score = 1.0 / (1.0 + np.exp(-x))
    else:
        score = np.exp(x - x.max(1, keepdims=True))
        score /= score.sum(1, keepdims=True)
    choice = score + (0.0 if inp["bias"] is None else inp["bias"].cpu().numpy().astype(np.float64))
    per = np.sort(choice.reshape(T, G, size), axis=2)
    best = per[..., -1].copy()
    if case["group_score"] == "top2" and size > 1:
        best += per[..., -2]
    group_rank = np.argsort(np.argsort(-best, axis=1, kind="stable"), axis=1, kind="stable")
    out = np.repeat(group_rank >= case["keep"], size, axis=1)
    # experts that stay before those that do not, then the larger choice, then the lower id
    ids = np.lexsort((np.broadcast_to(np.arange(E), (T, E)), -choice, out), axis=1)[:, :k]
    w = np.take_along_axis(score, ids, 1)
    if case["renormalise"]:
        w = w / w.sum(1, keepdims=True)
    w = w * np.float64(np.float32(case["scale"]))
    if case["shared"]:
        dot = inp["h"].float().cpu().numpy().astype(np.float64) @ inp["gate"].float().cpu().numpy().astype(np.float64)
        ids = np.concatenate([ids, np.full((T, 1), E)], axis=1)
        w = np.concatenate([w, (1.0 / (1.0 + np.exp(-dot)))[:, None]], axis=1)
    return torch.from_numpy(ids.astype(np.int32)), torch.from_numpy(w)


def _exact_sample(case, inp):
    logits = inp["logits"].float().cpu().numpy().astype(np.float64)
    u = inp["u"].cpu().numpy().astype(np.float64)
    B, V = logits.shape
    setting = {}
    for key in ("temperature", "top_k", "top_p", "min_p"):
        v = inp[key]
        v = v.cpu().numpy() if torch.is_tensor(v) else np.full(B, v, dtype=np.int64 if key == "top_k" else np.float32)
        setting[key] = v.astype(np.int64 if key == "top_k" else np.float64)
    tokens, logprobs = np.empty(B, dtype=np.int64), np.empty(B)
    for b in range(B):
        row, t, k = logits[b], setting["temperature"][b], setting["top_k"][b]
        if t <= 0:
            tokens[b], logprobs[b] = int(np.argmax(row)), 0.0
            continue
        w = np.exp((row - row.max()) / t)
        order = np.argsort(-row, kind="stable")
        if 0 < k < V:
            order = order[:k]
        mass = w[order]
        if setting["top_p"][b] < 1:
            before = np.concatenate([[0.0], np.cumsum(mass)[:-1]])
            order = order[:max(1, int(np.searchsorted(before, setting["top_p"][b] * mass.sum(), side="left")))]
        order = np.sort(order[w[order] >= setting["min_p"][b]])
        run = np.cumsum(w[order])
        at = min(int(np.searchsorted(run, u[b] * run[-1], side="right")), len(order) - 1)
        tokens[b], logprobs[b] = order[at], np.log(w[order[at]] / run[-1])
    return torch.from_numpy(tokens), torch.from_numpy(logprobs)


def exact(case, seed):
    inp = _inputs(case, seed)
    return (_exact_route if case["kind"] == "route" else _exact_sample)(case, inp)
