"""FCs whose weights depend on the row, as measurable cases: experts and low-rank adapters beside ``fc_Q4A``.

``route``   the router of a layer of experts: softmax over the experts, the best ``top_k`` of each token, and the plan
            that sorts the (token, slot) pairs by expert.
``up``      router, then the experts' product of the tokens: ``y[t, s] = fc_Q4A(x[t], W[ids[t, s]])``.
``down``    router, then the experts' product of a row per (token, slot), summed per token with the router's weights.
``lora``    a shared projection with an adapter per request: ``y = fc_Q4A(x) + scale[i] * B[i] (A[i] x)``.

Every FC quantizes its input as ``fc_Q4A`` does: per group of ``group_k`` values of a row, d = max|x| / 127, codes
round(x / d) in fp32 arithmetic (by definition: a code is a whole number that a rounding decides), group sums of the raw
values for the minima of Q4_1.  A row without an expert (id -1) gives zeros, a request without an adapter the shared
projection alone.

With ``own`` false the operators are computed by elementary torch operations in fp32, with it by this package.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

WIDE = (4096, 11008)       # hidden and intermediate width of the decode benchmark's model
MOST_WORK = 2 * 4096 * 22016 * 4096   # operations of the largest experts' product (2048 tokens, two experts each)


def listed() -> list[dict]:
    return [
        # one token through a router of few experts: the smallest call, all latency
        dict(name="route_1tok", kind="route", tokens=1, experts=8, top_k=2, renormalize=True, masked=False),
        # a long prompt through a router of many experts, some of them closed to some tokens
        dict(name="route_4096tok", kind="route", tokens=4096, experts=128, top_k=8, renormalize=False, masked=True),
        # one generated token through gate and up of two wide experts
        dict(name="up_1tok_wide", kind="up", tokens=1, experts=8, top_k=2, K=4096, N=22016, qtype="q4_1", group_k=32,
             masked=False),
        # eight sequences decoding together, many narrow experts
        dict(name="up_8tok_narrow", kind="up", tokens=8, experts=64, top_k=6, K=2048, N=2816, qtype="q4_1", group_k=128,
             masked=False),
        # a short prompt, sizes that fit no tile, experts with few rows each, some tokens closed to all experts
        dict(name="up_333tok_ragged", kind="up", tokens=333, experts=64, top_k=4, K=2001, N=1003, qtype="q4_0",
             group_k=32, masked=True),
        # a prompt of 2048 tokens through gate and up of wide experts: the largest product
        dict(name="up_2048tok_wide", kind="up", tokens=2048, experts=8, top_k=2, K=4096, N=22016, qtype="q4_1",
             group_k=128, masked=False),
        # one generated token back through the down projections of two wide experts
        dict(name="down_1tok_wide", kind="down", tokens=1, experts=8, top_k=2, K=11008, N=4096, qtype="q4_1",
             group_k=128, masked=False),
        # a batch of sequences and a prompt's end together: sixteen rows for each of many narrow experts
        dict(name="down_170tok_narrow", kind="down", tokens=170, experts=64, top_k=6, K=1408, N=2048, qtype="q4_1",
             group_k=32, masked=True),
        # eight requests decoding together, each with an adapter of its own
        dict(name="lora_8rows", kind="lora", rows=8, runs=8, adapters=16, rank=16, K=4096, N=4096, qtype="q4_1",
             group_k=32, dtype="bf16"),
        # many requests decoding together, some without an adapter
        dict(name="lora_61rows", kind="lora", rows=61, runs=61, adapters=40, rank=64, K=4096, N=11008, qtype="q4_1",
             group_k=128, dtype="fp16"),
        # a few short prompts, odd sizes, adapters kept in fp32
        dict(name="lora_ragged_fp32", kind="lora", rows=133, runs=5, adapters=3, rank=12, K=1001, N=2999, qtype="q4_0",
             group_k=32, dtype="fp32"),
        # prompts of several requests at once
        dict(name="lora_2048rows", kind="lora", rows=2048, runs=6, adapters=4, rank=32, K=4096, N=4096, qtype="q4_1",
             group_k=128, dtype="bf16"),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _size(rng, lo: int, hi: int) -> int:
    """A width: half of them multiples of 128, as model widths are, the others anything."""
    v = _log(rng, lo, hi)
    return max(128, v // 128 * 128) if rng.random() < 0.5 else v


def draw(rng) -> dict:
    kind = rng.choice(("route", "up", "down", "lora"))
    if kind == "route":
        experts = _log(rng, 2, 256)
        return dict(kind=kind, tokens=_log(rng, 1, 4096), experts=experts, top_k=rng.randint(1, min(8, experts)),
                    renormalize=rng.random() < 0.5, masked=rng.random() < 0.3)
    block = dict(qtype=rng.choice(("q4_0", "q4_1")), group_k=rng.choice((32, 128)))
    if kind == "lora":
        rows = _log(rng, 1, 2048)
        return dict(kind=kind, rows=rows, runs=min(rows, _log(rng, 1, 64)), adapters=_log(rng, 1, 64),
                    rank=rng.choice((4, 8, 16, 24, 32, 64, 128)), K=_size(rng, 256, 8192), N=_size(rng, 256, 11008),
                    dtype=rng.choice(("bf16", "fp16", "fp32")), **block)
    experts = _log(rng, 2, 128)
    top_k = rng.randint(1, min(8, experts))
    tokens = _log(rng, 1, 2048)
    K, N = _size(rng, 256, 8192), _size(rng, 256, 8192)
    while experts * K * N > 8 * 4096 * 22016 or experts * tokens * top_k * N * K * 2 > 4 * MOST_WORK:
        if experts * K * N > 8 * 4096 * 22016:
            K, N = max(256, K // 2), max(256, N // 2)
        else:
            tokens = max(1, tokens // 2)
    return dict(kind=kind, tokens=tokens, experts=experts, top_k=top_k, K=K, N=N, masked=rng.random() < 0.3, **block)


# ------------------------------------------------------------------------------------------------ inputs
def _weights(shape: tuple[int, ...], qtype: str, group_k: int, g: torch.Generator) -> torch.Tensor:
    """Packed weights as the packer leaves them of N(0, 0.02): nibbles about the middle level, fp16 scales, minima."""
    levels = torch.randn(*shape, 16 * group_k, 2, device="cuda", generator=g, dtype=torch.float16)
    levels = levels.mul_(3.0).add_(7.5).round_().clamp_(0, 15).to(torch.uint8)
    body = levels[..., 0] | (levels[..., 1] << 4)
    d = (torch.rand(*shape, 32, device="cuda", generator=g) * 0.3 + 0.85) * 0.0065
    parts = [body, d.half().view(torch.uint8)]
    if qtype == "q4_1":
        m = d * -(torch.rand(*shape, 32, device="cuda", generator=g) + 7.0)
        parts.append(m.half().view(torch.uint8))
    return torch.cat(parts, -1).view(torch.int8)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator("cuda").manual_seed(seed)
    kind = case["kind"]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if kind == "lora":
        rows, K, N, r, n = case["rows"], case["K"], case["N"], case["rank"], case["adapters"]
        dtype = dict(bf16=torch.bfloat16, fp16=torch.float16, fp32=torch.float32)[case["dtype"]]
        # requests one after the other, of ragged lengths; one in eight has no adapter
        edges = torch.rand(case["runs"] - 1, device="cuda", generator=g).sort().values
        if case["runs"] == rows:
            edges = torch.arange(1, rows, device="cuda") / rows
        request = torch.searchsorted(edges, (torch.arange(rows, device="cuda") + 0.5) / rows)
        of_request = torch.randint(0, n, (case["runs"],), device="cuda", generator=g)
        of_request[torch.rand(case["runs"], device="cuda", generator=g) < 0.125] = -1
        shape = (-(-N // 32), -(-K // case["group_k"]))
        return dict(case=case, x=randn(1, rows, K), ids=of_request[request].to(torch.int32).view(1, rows),
                    wq=_weights(shape, case["qtype"], case["group_k"], g), a=(randn(n, r, K) / math.sqrt(K)).to(dtype),
                    b=(randn(n, N, r) * 0.02).to(dtype), scales=torch.rand(n, device="cuda", generator=g) + 1.0)
    T, E = case["tokens"], case["experts"]
    logits = randn(1, T, E) * 1.5
    if case["masked"]:
        # experts closed to a token (a quarter of them), and a few padding tokens without any
        logits[torch.rand(1, T, E, device="cuda", generator=g) < 0.25] = -math.inf
        logits[torch.rand(1, T, device="cuda", generator=g) < 0.03] = -math.inf
    state = dict(case=case, logits=logits)
    if kind != "route":
        shape = (E, -(-case["N"] // 32), -(-case["K"] // case["group_k"]))
        state["wq"] = _weights(shape, case["qtype"], case["group_k"], g)
        state["x"] = randn(1, T, case["K"]) if kind == "up" else randn(1, T, case["top_k"], case["K"])
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_route(logits: torch.Tensor, k: int, renormalize: bool):
    E = logits.shape[-1]
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    best, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
    closed = best[..., :k] == -math.inf
    chosen = torch.gather(p, -1, ids[..., :k])
    total = chosen.sum(-1, keepdim=True) if renormalize else total
    weights = torch.where(closed, torch.zeros_like(chosen), chosen / total)
    ids = torch.where(closed, -1, ids[..., :k]).to(torch.int32)
    # the pairs sorted by expert, those without one behind the others; where each expert's pairs begin
    flat = ids.reshape(-1).to(torch.int64)
    key, order = torch.sort(torch.where(flat < 0, E, flat), stable=True)
    offsets = torch.searchsorted(key, torch.arange(E + 1, device=key.device))
    return weights, ids, offsets.to(torch.int32), order.to(torch.int32)


def _plain_quantize(x: torch.Tensor, G: int):
    """fp32 [rows, K] -> what the codes stand for [rows, Kg * G], group sums [rows, Kg]."""
    rows, K = x.shape
    Kg = -(-K // G)
    v = torch.nn.functional.pad(x, (0, Kg * G - K)).view(rows, Kg, G)
    d = v.abs().amax(-1, keepdim=True) / torch.full((1,), 127.0, device=x.device)  # (a tensor: torch divides by it)
    t = v * torch.where(d == 0, torch.zeros_like(d), torch.reciprocal(d))
    code = torch.round(t)
    body = K // 8 * 8  # values behind the last whole eight round half away from zero
    away = (torch.sign(t) * torch.floor(t.abs().double() + 0.5)).float()
    k = torch.arange(Kg * G, device=x.device).view(Kg, G)
    code = torch.where((k >= body) & (k < K), away, code).clamp(-128, 127)
    return (code * d).view(rows, Kg * G), v.sum(-1)


def _plain_unpack(wq: torch.Tensor, qtype: str, G: int):
    """packed [..., Ng, Kg, bytes] -> fp32 [..., Ng * 32, Kg * G] without the minima, minima [..., Ng * 32, Kg]."""
    lead, (Ng, Kg) = wq.shape[:-3], wq.shape[-3:-1]
    u = wq.view(torch.uint8)
    body = u[..., : 16 * G].reshape(*lead, Ng, Kg, G // 8, 32, 4)
    d = u[..., 16 * G: 16 * G + 64].contiguous().view(torch.float16).float()
    nibbles = torch.stack((body & 15, body >> 4), -2).float()  # [.., Ng, Kg, G/8, column, half, 4]
    nibbles *= d.view(*lead, Ng, Kg, 1, 32, 1, 1)
    dims = len(lead)
    w = nibbles.permute(*range(dims), dims, dims + 3, dims + 1, dims + 2, dims + 4, dims + 5)
    w = w.reshape(*lead, Ng * 32, Kg * G)
    if qtype == "q4_0":
        return w, None
    m = u[..., 16 * G + 64:].contiguous().view(torch.float16).float()
    return w, m.transpose(-1, -2).reshape(*lead, Ng * 32, Kg)


def _plain_fc(x: torch.Tensor, wq: torch.Tensor, N: int, qtype: str, G: int) -> torch.Tensor:
    """fp32 [rows, K] through packed weights [..., Ng, Kg, bytes] -> [..., rows, N]."""
    values, sums = _plain_quantize(x, G)
    w, m = _plain_unpack(wq, qtype, G)
    y = values @ w.transpose(-1, -2)
    if m is not None:
        y += sums @ m.transpose(-1, -2)
    return y[..., :N]


def _plain_experts(state: dict):
    c = state["case"]
    T, k, N = c["tokens"], c["top_k"], c["N"]
    weights, ids, _, _ = _plain_route(state["logits"], k, True)
    of = ids.view(T, k).to(torch.int64)
    rows = state["x"].reshape(-1, c["K"])  # a row per token, or per (token, slot)
    every = _plain_fc(rows, state["wq"], N, c["qtype"], c["group_k"])  # of every expert
    row = torch.arange(rows.shape[0], device=rows.device).view(T, -1).expand(T, k)
    y = torch.where((of < 0)[..., None], 0.0, every[of.clamp(min=0), row])
    if c["kind"] == "down":
        y = (y * weights.view(T, k, 1)).sum(1)
    return dict(weights=weights, ids=ids, y=y[None])


def _plain_lora(state: dict) -> torch.Tensor:
    c = state["case"]
    x, ids = state["x"][0], state["ids"][0].to(torch.int64)
    y = _plain_fc(x, state["wq"], c["N"], c["qtype"], c["group_k"])
    mine = (ids == torch.arange(c["adapters"], device=ids.device)[:, None]) * state["scales"][:, None]
    t = (x @ state["a"].float().transpose(-1, -2)) * mine[..., None]                # [adapters, rows, rank]
    n, rows, r = t.shape
    y = y + t.transpose(0, 1).reshape(rows, n * r) @ state["b"].float().transpose(-1, -2).reshape(n * r, c["N"])
    return y[None]


# ------------------------------------------------------------------------------------------------ a pass
def run(state: dict):
    c = state["case"]
    if own:
        from llama_cl_b200 import llmops

        if c["kind"] == "lora":
            groups = llmops.group_rows(state["ids"], c["adapters"])
            return llmops.fc_Q4A_lora(state["x"], state["wq"], c["N"], state["a"], state["b"], groups,
                                      scales=state["scales"])
        if c["kind"] == "route":
            weights, groups = llmops.route_top_k(state["logits"], c["top_k"], renormalize=c["renormalize"])
            return dict(weights=weights, ids=groups.ids, offsets=groups.offsets, order=groups.order)
        weights, groups = llmops.route_top_k(state["logits"], c["top_k"])
        y = llmops.fc_Q4A_experts(state["x"], state["wq"], c["N"], groups,
                                  weights=weights if c["kind"] == "down" else None)
        return dict(weights=weights, ids=groups.ids, y=y)
    if c["kind"] == "lora":
        return _plain_lora(state)
    if c["kind"] == "route":
        weights, ids, offsets, order = _plain_route(state["logits"], c["top_k"], c["renormalize"])
        return dict(weights=weights, ids=ids, offsets=offsets, order=order)
    return _plain_experts(state)


def work(case: dict) -> dict:
    if case["kind"] == "route":
        T, E, k = case["tokens"], case["experts"], case["top_k"]
        return dict(bytes=4 * (T * E + 3 * T * k + E + 1), flops=4 * T * E)
    K, N, G = case["K"], case["N"], case["group_k"]
    packed = -(-N // 32) * -(-K // G) * (16 * G + (128 if case["qtype"] == "q4_1" else 64))
    if case["kind"] == "lora":
        rows, r = case["rows"], case["rank"]
        used = case["adapters"] * (1 - (1 - 1 / case["adapters"]) ** (case["runs"] * 0.875))
        each = 4 if case["dtype"] == "fp32" else 2
        return dict(bytes=packed + 4 * rows * (K + N) + used * each * r * (K + N),
                    flops=2 * rows * K * N + 2 * 0.875 * rows * r * (K + N))
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    pairs = T * k
    used = E * (1 - (1 - k / E) ** T)  # experts that at least one token takes
    rows_in, rows_out = (T, pairs) if case["kind"] == "up" else (pairs, T)
    return dict(bytes=used * packed + 4 * (rows_in * K + rows_out * N + T * E), flops=2 * pairs * K * N)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_fc(x: np.ndarray, wq: torch.Tensor, N: int, qtype: str, G: int) -> torch.Tensor:
    """One weight tensor: fp32 rows [rows, K], packed [Ng, Kg, bytes] -> float64 [rows, N] on the GPU."""
    rows, K = x.shape
    Ng, Kg, _ = wq.shape
    codes, scales, sums = np.zeros((rows, Kg * G), np.float64), np.zeros((rows, Kg)), np.zeros((rows, Kg))
    for kb in range(Kg):
        part = x[:, kb * G: (kb + 1) * G]
        d = np.abs(part).max(1) / np.float32(127)
        inverse = np.divide(np.float32(1), d, out=np.zeros_like(d), where=d != 0)
        t = part * inverse[:, None]  # fp32: the definition of a code
        q = np.rint(t).astype(np.float64)
        body = part.shape[1] // 8 * 8
        q[:, body:] = np.trunc(t[:, body:].astype(np.float64) + np.copysign(0.5, t[:, body:]))
        codes[:, kb * G: kb * G + part.shape[1]] = np.clip(q, -128, 127)
        scales[:, kb], sums[:, kb] = d, part.astype(np.float64).sum(1)
    codes, scales, sums = (torch.from_numpy(v).cuda() for v in (codes, scales, sums))
    u = wq.view(torch.uint8)
    y = torch.zeros(rows, Ng * 32, dtype=torch.float64, device="cuda")
    step = max(1, 2048 // G)
    for k0 in range(0, Kg, step):
        blocks = u[:, k0: k0 + step]
        n = blocks.shape[1]
        word = blocks[..., : 16 * G].reshape(Ng, n, G // 8, 32, 4)
        w = torch.empty(Ng, 32, n, G // 8, 8, dtype=torch.float64, device="cuda")
        w[..., :4] = (word & 15).permute(0, 3, 1, 2, 4)
        w[..., 4:] = (word >> 4).permute(0, 3, 1, 2, 4)
        d = blocks[..., 16 * G: 16 * G + 64].contiguous().view(torch.float16).double()  # [Ng, n, 32]
        w *= d.permute(0, 2, 1)[..., None, None]
        a = codes[:, k0 * G: (k0 + n) * G].view(rows, n, G) * scales[:, k0: k0 + n, None]
        y += a.view(rows, n * G) @ w.view(Ng * 32, n * G).t()
        if qtype == "q4_1":
            m = blocks[..., 16 * G + 64:].contiguous().view(torch.float16).double()
            y += sums[:, k0: k0 + n] @ m.permute(0, 2, 1).reshape(Ng * 32, n).t()
    return y[:, :N]


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "lora":
        ids, x = s["ids"][0].cpu().numpy(), s["x"][0]
        y = _exact_fc(x.cpu().numpy(), s["wq"], case["N"], case["qtype"], case["group_k"])
        for i in np.unique(ids[ids >= 0]).tolist():
            rows = torch.from_numpy(np.nonzero(ids == i)[0]).cuda()
            t = x[rows].double() @ s["a"][i].double().t()
            y[rows] += s["scales"][i].double() * (t @ s["b"][i].double().t())
        return y[None]
    logits, k = s["logits"][0].double().cpu().numpy(), case["top_k"]
    T, E = logits.shape
    weights, ids = np.zeros((T, k)), np.full((T, k), -1, np.int64)
    for t in range(T):
        finite = logits[t] > -math.inf
        if not finite.any():
            continue
        p = np.where(finite, np.exp(logits[t] - logits[t][finite].max()), 0.0)
        best = sorted((e for e in range(E) if finite[e]), key=lambda e: (-logits[t, e], e))[:k]
        ids[t, : len(best)] = best
        total = p[best].sum() if case.get("renormalize", True) else p.sum()
        weights[t, : len(best)] = p[best] / total
    out = dict(weights=weights[None], ids=ids[None])
    if case["kind"] == "route":
        return out | dict(offsets=None, order=None)
    N = case["N"]
    y = torch.zeros(T, k, N, dtype=torch.float64, device="cuda")
    x = s["x"][0].cpu().numpy()
    for e in np.unique(ids[ids >= 0]).tolist():
        t, slot = np.nonzero(ids == e)
        rows = x[t] if case["kind"] == "up" else x[t, slot]
        y[torch.from_numpy(t).cuda(), torch.from_numpy(slot).cuda()] = _exact_fc(rows, s["wq"][e], N, case["qtype"],
                                                                                  case["group_k"])
    if case["kind"] == "down":
        y = (y * torch.from_numpy(weights).cuda()[..., None]).sum(1)
    return out | dict(y=y[None])
