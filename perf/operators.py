"""Operators of a serving step over a paged cache, as a user calls them, beside their plain forms:

  append     queries and keys normed per head, rotated, and keys and values appended to a paged cache
  attention  chunks of new tokens (one token to whole prompts) over a paged cache
  adapters   low-rank adapters of many requests beside a shared projection

`own` false: elementary torch operations in 32 bits.  `own` true: the package's calls.
"""
from __future__ import annotations

import functools
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
EPS = 1e-5


@functools.lru_cache(None)
def _extension():
    name = "llama3_custom_inference_b200"
    if name not in sys.modules:
        folder = Path(__file__).resolve().parent.parent / "llama3-custom-inference_b200"
        spec = importlib.util.spec_from_file_location(name, folder / "__init__.py", submodule_search_locations=[str(folder)])
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return sys.modules[name].extension()


# ---- the cases -----------------------------------------------------------------------------------------------------
# append and attention: B sequences, `chunks` of them with up to T new tokens and the others with one, up to S tokens with
# the new ones; ragged: sequences of different lengths.  adapters: `rows` tokens in runs of `run` of one request.
def listed() -> list:
    return [
        # a decode step of a full serving batch
        {"name": "append_step", "kind": "append", "B": 64, "Hq": 32, "Hkv": 8, "D": 128, "page": 16, "S": 512, "T": 1, "chunks": 0, "ragged": True, "norms": False},
        # one prompt of odd length of a model with norms of queries and keys
        {"name": "append_prompt", "kind": "append", "B": 1, "Hq": 24, "Hkv": 8, "D": 64, "page": 48, "S": 2001, "T": 2001, "chunks": 1, "ragged": False, "norms": True},
        # chunks of many prompts in one pass
        {"name": "append_chunks", "kind": "append", "B": 24, "Hq": 64, "Hkv": 8, "D": 128, "page": 32, "S": 1500, "T": 500, "chunks": 20, "ragged": True, "norms": True},
        # one chat sequence at the start of its answer: latency
        {"name": "step_short", "kind": "attention", "B": 1, "Hq": 32, "Hkv": 8, "D": 64, "page": 16, "S": 257, "T": 1, "chunks": 0, "ragged": False},
        # a serving batch whose sequences are at different lengths
        {"name": "step_ragged", "kind": "attention", "B": 16, "Hq": 64, "Hkv": 8, "D": 128, "page": 16, "S": 8000, "T": 1, "chunks": 0, "ragged": True},
        # one sequence behind a whole book
        {"name": "step_long", "kind": "attention", "B": 1, "Hq": 32, "Hkv": 8, "D": 128, "page": 64, "S": 131072, "T": 1, "chunks": 0, "ragged": False},
        # the next chunk of two long documents
        {"name": "chunk", "kind": "attention", "B": 2, "Hq": 32, "Hkv": 8, "D": 128, "page": 16, "S": 16500, "T": 512, "chunks": 2, "ragged": False},
        # a step of a server: two prompts' chunks beside the answers of other requests
        {"name": "mixed", "kind": "attention", "B": 12, "Hq": 32, "Hkv": 8, "D": 128, "page": 32, "S": 4100, "T": 400, "chunks": 2, "ragged": True},
        # prompts read in from their first token
        {"name": "prompts", "kind": "attention", "B": 4, "Hq": 32, "Hkv": 8, "D": 64, "page": 32, "S": 2048, "T": 2048, "chunks": 4, "ragged": True},
        # a few answers at once, each of its own adapter
        {"name": "adapters_step", "kind": "adapters", "rows": 8, "K": 2048, "N": 8192, "rank": 16, "adapters": 8, "run": 1},
        # a full batch of answers, many adapters
        {"name": "adapters_batch", "kind": "adapters", "rows": 64, "K": 8192, "N": 2048, "rank": 32, "adapters": 40, "run": 1},
        # prompts of several requests in one pass
        {"name": "adapters_prompt", "kind": "adapters", "rows": 6001, "K": 2048, "N": 8192, "rank": 16, "adapters": 6, "run": 900},
    ]


def _log(rng, low, high) -> int:
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


HEADS = [(32, 8), (24, 8), (64, 8), (16, 4), (32, 4), (16, 1)]


def draw(rng) -> dict:
    kind = rng.choice(["append", "append", "attention", "attention", "attention", "attention", "adapters", "adapters"])
    if kind == "adapters":
        rows = _log(rng, 1, 6000)
        K, N = 8 * _log(rng, 64, 1024), 8 * _log(rng, 32, 1024)
        if rows * K * N > 6001 * 2048 * 8192:
            K = N = 2048
        return {"kind": kind, "rows": rows, "K": K, "N": N, "rank": rng.choice([8, 16, 32, 40, 64, 128]), "adapters": _log(rng, 1, 64),
                "run": 1 if rows <= 64 else _log(rng, 64, rows)}
    Hq, Hkv = rng.choice(HEADS)
    D, page = rng.choice([64, 128]), rng.choice([16, 32, 48, 64, 128, 256])
    if kind == "append":
        B = _log(rng, 1, 64)
        T = _log(rng, 1, 8000 // B)
        return {"kind": kind, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "S": T + _log(rng, 1, 8000 // B), "T": T,
                "chunks": rng.choice([0, B, rng.randint(0, B)]), "ragged": rng.random() < 0.5, "norms": rng.random() < 0.5}
    if rng.random() < 0.5:   # a decode step
        B = _log(rng, 1, 64)
        return {"kind": kind, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "S": _log(rng, 16, 131072 // B), "T": 1, "chunks": 0,
                "ragged": rng.random() < 0.5}
    B = rng.randint(1, 8)
    T = _log(rng, 2, 2048 // B)
    case = {"kind": kind, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "S": T + _log(rng, 1, 16000 // B), "T": T,
            "chunks": rng.choice([B, rng.randint(1, B)]), "ragged": rng.random() < 0.5}
    while work(case)["flops"] > 2.7e11:   # (the largest listed one)
        case["T"] //= 2
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _lengths(case):
    """New tokens and tokens with them of every sequence: of the case alone, so that its work is the same for every seed."""
    new, total = [], []
    for b in range(case["B"]):
        share = 1 - 0.6 * (b * 0.6180339887 % 1) if case["ragged"] else 1.0
        n = max(1, round(case["T"] * share)) if b < case["chunks"] else 1
        before = round((case["S"] - case["T"]) * share)
        new.append(n)
        total.append(before + n)
    return new, total


def _runs(case):
    """Adapter of every row: runs of one request, every seventh request without an adapter."""
    requests = [r // case["run"] for r in range(case["rows"])]
    return [-1 if q % 7 == 6 else q * 5 % case["adapters"] for q in requests]


def _uniform(case):
    """New tokens per sequence where all have the same number, and a batch is [B, T, ...]; else 0, and tokens lie one behind the other."""
    new, _ = _lengths(case)
    return new[0] if min(new) == max(new) else 0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0, dtype=BF16):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def near_one(n):
        return (1.0 + 0.1 * torch.randn(n, generator=g, device="cuda")).to(BF16)

    state = {"case": case}
    if case["kind"] == "adapters":
        K, N, rank, n = case["K"], case["N"], case["rank"], case["adapters"]
        state.update(x=randn(case["rows"], K), w=randn(N, K, scale=K ** -0.5), a=randn(n, rank, K, scale=K ** -0.5),
                     b=randn(n, N, rank, scale=rank ** -0.5),
                     scales=0.5 + torch.rand(n, generator=g, device="cuda"),
                     index=torch.tensor(_runs(case), dtype=torch.int32, device="cuda"))
        return state
    B, Hq, Hkv, D, page = (case[k] for k in ("B", "Hq", "Hkv", "D", "page"))
    new, total = _lengths(case)
    T, N = _uniform(case), sum(new)
    need = [-(-t // page) for t in total]
    # pages in any order, as a server hands them out
    order = torch.randperm(sum(need) + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(B, max(need), dtype=torch.int32, device="cuda")
    first = 0
    for b, n in enumerate(need):
        table[b, :n] = order[first:first + n]
        first += n
    starts = torch.zeros(B + 1, dtype=torch.int64)
    starts[1:] = torch.tensor(new).cumsum(0)
    state.update(T=T, longest=max(new), table=table, starts=starts.to(torch.int32).cuda(),
                 seq_lens=torch.tensor(total, dtype=torch.int32, device="cuda"),
                 positions=torch.tensor([t - n for t, n in zip(total, new)], dtype=torch.int32, device="cuda"),
                 cache_k=randn(len(order), page, Hkv, D), cache_v=randn(len(order), page, Hkv, D))
    if case["kind"] == "attention":
        state["q"] = randn(N, Hq, D).view(*((B, T) if T else (N,)), Hq, D)
        return state
    width = (Hq + 2 * Hkv) * D
    state["qkv"] = randn(N, width).view(*((B, T) if T else (N,)), width)
    angles = torch.arange(max(total), dtype=F64, device="cuda")[:, None] * 500000.0 ** (-torch.arange(0, D, 2, dtype=F64, device="cuda") / D)
    state["freq"] = torch.stack([angles.cos(), angles.sin()], dim=-1).reshape(max(total), D).to(F32)
    state["q_norm"], state["k_norm"] = (near_one(D), near_one(D)) if case["norms"] else (None, None)
    return state


# ---- plain forms ----------------------------------------------------------------------------------------------------
def _rows(s, n_rows):
    """Sequence and place among its new tokens of every row."""
    row = torch.arange(n_rows, device="cuda")
    starts = s["starts"].long()
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    return seq, row - starts[seq]


def _append(s):
    c = s["case"]
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    qkv = s["qkv"].float().view(-1, Hq + 2 * Hkv, D)
    q, k, v = qkv.split([Hq, Hkv, Hkv], dim=1)
    seq, t = _rows(s, qkv.shape[0])
    pos = s["positions"].long()[seq] + t
    if s["q_norm"] is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"].float()
    turn = s["freq"][pos].view(-1, 1, D // 2, 2)
    cos, sin = turn[..., 0], turn[..., 1]

    def rotate(x):
        x = x.unflatten(-1, (D // 2, 2))
        return torch.stack([x[..., 0] * cos - x[..., 1] * sin, x[..., 0] * sin + x[..., 1] * cos], dim=-1).flatten(-2).to(BF16)

    page = s["table"].long()[seq, pos // c["page"]]
    s["cache_k"][page, pos % c["page"]] = rotate(k)
    s["cache_v"][page, pos % c["page"]] = v.to(BF16)
    return rotate(q).view(*s["qkv"].shape[:-1], Hq, D)


def _attention(s):
    c = s["case"]
    B, Hq, Hkv, D, T = c["B"], c["Hq"], c["Hkv"], c["D"], s["longest"]
    R = Hq // Hkv
    q = s["q"].reshape(-1, Hq, D)
    starts, lens = s["starts"].long(), s["seq_lens"].long()
    place = starts[:-1, None] + torch.arange(T, device="cuda")                                 # [B, T], padded at the end of a sequence
    pos = (lens - starts[1:])[:, None] + place
    qp = q[place.clamp(max=q.shape[0] - 1)].float().view(B, T, Hkv, R, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, R * T, D)
    table = s["table"].long()
    k = s["cache_k"][table].float().flatten(1, 2).permute(0, 2, 3, 1)                          # [B, Hkv, D, S]
    v = s["cache_v"][table].float().flatten(1, 2).transpose(1, 2)                              # [B, Hkv, S, D]
    score = (qp @ k * D ** -0.5).view(B, Hkv, R, T, -1)
    unseen = torch.arange(k.shape[-1], device="cuda") > pos[:, :, None]
    score = score.masked_fill_(unseen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = (p.flatten(2, 3) @ v).view(B, Hkv, R, T, D) / p.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(BF16)
    return o[place < starts[1:, None]].view(s["q"].shape)


def _adapters(s):
    rows, (n, rank, K) = s["x"].shape[0], s["a"].shape
    x, index = s["x"].float(), s["index"].long()
    z = (x @ s["a"].float().view(n * rank, K).T).view(rows, n, rank)
    mine = torch.arange(n, device="cuda") == index[:, None]                                     # one adapter's part of z, or none
    z = torch.where(mine[..., None], z * s["scales"][:, None], 0.0).view(rows, n * rank)
    return (x @ s["w"].float().T + z @ s["b"].float().transpose(1, 2).reshape(n * rank, -1)).to(BF16)


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if c["kind"] == "adapters":
        if own:
            return _extension().adapter_linear(s["x"], s["w"], s["a"], s["b"], s["index"], scales=s["scales"])
        return _adapters(s)
    starts = None if s["T"] else s["starts"]
    if c["kind"] == "attention":
        if own:
            return _extension().paged_attention(s["q"], s["cache_k"], s["cache_v"], s["table"], s["seq_lens"], starts=starts)
        return _attention(s)
    if own:
        q = _extension().rot_embed_paged_kv_cache(s["qkv"], s["freq"], s["cache_k"], s["cache_v"], s["table"], s["positions"], c["Hq"], c["Hkv"],
                                                  starts=starts, q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
    else:
        q = _append(s)
    return {"q": q, "cache_k": s["cache_k"], "cache_v": s["cache_v"]}


def work(case) -> dict:
    if case["kind"] == "adapters":
        rows, K, N, rank = case["rows"], case["K"], case["N"], case["rank"]
        index = _runs(case)
        used, with_one = len(set(index) - {-1}), sum(i >= 0 for i in index)
        return {"bytes": 2 * (rows * K + N * K + rows * N + used * rank * (K + N)) + 4 * rows,
                "flops": 2 * rows * K * N + 2 * with_one * rank * (K + N)}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    new, total = _lengths(case)
    if case["kind"] == "append":
        N = sum(new)
        return {"bytes": 4 * N * (Hq + 2 * Hkv) * D + 4 * D * len({p for n, t in zip(new, total) for p in range(t - n, t)}), "flops": 8 * N * (Hq + Hkv) * D}
    seen = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))                     # visible (token, key) pairs
    return {"bytes": 4 * sum(total) * Hkv * D + 4 * sum(new) * Hq * D, "flops": 4 * seen * Hq * D}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "adapters":
        x, index = s["x"].to(F64), _runs(case)
        y = torch.empty(case["rows"], case["N"], dtype=F64, device="cuda")
        for i in set(index):
            at = torch.tensor([r for r, v in enumerate(index) if v == i], device="cuda")
            y[at] = torch.mm(x[at], s["w"].to(F64).t())
            if i >= 0:
                y[at] += float(s["scales"][i]) * torch.mm(torch.mm(x[at], s["a"][i].to(F64).t()), s["b"][i].to(F64).t())
        return y
    new, total = _lengths(case)
    Hq, Hkv, D, page = case["Hq"], case["Hkv"], case["D"], case["page"]
    table = s["table"].tolist()
    first = 0
    if case["kind"] == "append":
        tokens = s["qkv"].to(F64).reshape(sum(new), Hq + 2 * Hkv, D)
        q_out = torch.empty(sum(new), Hq, D, dtype=F64, device="cuda")
        ck, cv = s["cache_k"].to(F64), s["cache_v"].to(F64)
        for b, (n, end) in enumerate(zip(new, total)):
            mine = tokens[first:first + n]
            at = torch.arange(end - n, end, device="cuda")
            turn = torch.view_as_complex(s["freq"].to(F64)[at].reshape(n, 1, D // 2, 2).contiguous())
            parts = []
            for heads, weight in ((mine[:, :Hq], s["q_norm"]), (mine[:, Hq:Hq + Hkv], s["k_norm"])):
                if weight is not None:
                    heads = heads / (heads.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * weight.to(F64)
                pairs = torch.view_as_complex(heads.reshape(n, -1, D // 2, 2).contiguous())
                parts.append(torch.view_as_real(pairs * turn).reshape(n, -1, D))
            q_out[first:first + n] = parts[0]
            flat = torch.tensor(table[b], device="cuda")[at // page] * page + at % page
            ck.view(-1, Hkv, D)[flat] = parts[1]
            cv.view(-1, Hkv, D)[flat] = mine[:, Hq + Hkv:]
            first += n
        return {"q": q_out.view(*s["qkv"].shape[:-1], Hq, D), "cache_k": ck, "cache_v": cv}
    if sum(n * t for n, t in zip(new, total)) * Hq * D > 4e11:    # (minutes in 64 bits)
        return None
    out = torch.empty(sum(new), Hq, D, dtype=F64, device="cuda")
    q = s["q"].reshape(sum(new), Hq, D)
    for b, (n, end) in enumerate(zip(new, total)):
        pages = table[b][:-(-end // page)]
        k = s["cache_k"][pages].flatten(0, 1)[:end]
        v = s["cache_v"][pages].flatten(0, 1)[:end]
        for h in range(Hq):
            sc = q[first:first + n, h].to(F64) @ k[:, h * Hkv // Hq].to(F64).t() / math.sqrt(D)
            sc = torch.where(torch.ones(n, end, dtype=torch.bool, device="cuda").tril(end - n), sc, -math.inf)
            out[first:first + n, h] = torch.softmax(sc, dim=-1) @ v[:, h * Hkv // Hq].to(F64)
        first += n
    return out.view(s["q"].shape)
