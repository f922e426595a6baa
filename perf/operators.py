"""Attention over parts of a paged cache, and the joining of the parts: the operators' cases, their
plain forms in elementary torch operations and their definitions in 64 bits.

Families:
  shared   attention of a batch whose requests share long prefixes. Requests come in groups; a group's
           prefix is cached once, each request's own tokens (its suffix) follow on pages of its own. A
           query token sees its group's whole prefix and its request's suffix up to itself.
  window   attention in a sliding window whose first cached tokens stay visible: the query at
           position p sees t <= p with t >= p - window or t < first. One query token per request
           (new = 0 in the case: the decode form) or ragged runs of new ones.
  merge    the join of results computed over disjoint parts of a context, each with the base-2
           logarithm of its softmax mass.

Ragged lengths come from the case's own ``lens`` number, so the work of a case is known without its
inputs; values and page tables come from the seed given to ``prepare``.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16 = torch.bfloat16
WORKSPACE = 128 << 20  # the float workspace the wrappers are given
LOG2E = 1.4426950408889634

# heads of one layer: query heads, kv heads, head dim
HEADS = {
    "llama8b": (32, 8, 128),   # and Qwen3-8B
    "llama1b": (32, 8, 64),
    "oss": (64, 8, 64),        # gpt-oss
    "gemma": (16, 8, 256),
    "llama8b_tp4": (8, 2, 128),  # one rank's heads under four-way tensor parallelism
    "seven": (14, 2, 128),     # seven query heads per kv head
}


def listed():
    return [
        # a program's four branches from one short prompt: latency and launches
        {"name": "shared_4", "family": "shared", "model": "llama8b", "groups": 1, "batch": 4, "prefix_lo": 600,
         "prefix_hi": 600, "lo": 1, "hi": 60, "new": 0, "page": 16, "lens": 1},
        # several prompts at once, each decoded in a few beams; odd in every size
        {"name": "shared_beams", "family": "shared", "model": "llama8b", "groups": 9, "batch": 37, "prefix_lo": 300,
         "prefix_hi": 3500, "lo": 20, "hi": 400, "new": 0, "page": 16, "lens": 2},
        # an ordinary decode batch behind one system prompt, gpt-oss heads
        {"name": "shared_oss", "family": "shared", "model": "oss", "groups": 1, "batch": 61, "prefix_lo": 5000,
         "prefix_hi": 5000, "lo": 100, "hi": 1500, "new": 0, "page": 16, "lens": 3},
        # a full decode batch over one long document: the largest shared case
        {"name": "shared_256", "family": "shared", "model": "llama8b", "groups": 1, "batch": 256, "prefix_lo": 16000,
         "prefix_hi": 16000, "lo": 128, "hi": 1000, "new": 0, "page": 16, "lens": 4},
        # drafted tokens or short questions of many requests behind two prompts
        {"name": "shared_ragged", "family": "shared", "model": "llama8b", "groups": 2, "batch": 23, "prefix_lo": 2000,
         "prefix_hi": 5000, "lo": 1, "hi": 300, "new": 13, "page": 16, "lens": 5},
        # one long chat in a window that keeps its first tokens: latency
        {"name": "window_decode_1", "family": "window", "model": "llama8b", "batch": 1, "lo": 9000, "hi": 9000, "new": 0,
         "window": 1023, "first": 4, "lse": True, "page": 16, "lens": 6},
        # a full decode batch of streams in a window, mixed lengths (some shorter than the window)
        {"name": "window_decode_256", "family": "window", "model": "llama8b", "batch": 256, "lo": 128, "hi": 20000,
         "new": 0, "window": 2047, "first": 5, "lse": False, "page": 16, "lens": 7},
        # fresh prompts several windows long, prefilled at once: the largest case
        {"name": "window_prefill", "family": "window", "model": "llama8b", "batch": 5, "lo": 1500, "hi": 6000,
         "new": -1, "window": 1023, "first": 4, "lse": False, "page": 16, "lens": 8},
        # chunks of long streams (gpt-oss heads and window) that keep a 100-token instruction
        {"name": "window_chunk", "family": "window", "model": "oss", "batch": 4, "lo": 3000, "hi": 9000, "new": 500,
         "window": 127, "first": 100, "lse": True, "page": 16, "lens": 9},
        # two parts of a few decode rows
        {"name": "merge_2", "family": "merge", "states": 2, "tokens": 5, "heads": 32, "dim": 128, "dtype": "bf16"},
        # a long prompt's rows over four parts of its context
        {"name": "merge_4", "family": "merge", "states": 4, "tokens": 8190, "heads": 32, "dim": 128, "dtype": "bf16"},
        # partial results in fp32 from many pieces
        {"name": "merge_fp32", "family": "merge", "states": 17, "tokens": 300, "heads": 16, "dim": 256,
         "dtype": "fp32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    lens = rng.randrange(1 << 20)
    family = rng.choice(["shared", "shared", "shared", "window", "window", "merge"])
    model = rng.choice(["llama8b", "llama8b", "llama1b", "oss", "gemma", "llama8b_tp4", "seven"])
    page = rng.choice([16, 16, 16, 32, 5, 1])
    if family == "shared":
        batch = _log(rng, 1, 256)
        groups = min(batch, _log(rng, 1, 16))
        new = rng.choice([0, 0, 0, rng.randint(2, 24)])
        prefix = _log(rng, 20, min(16000, 64000 // groups, 4000000 // (batch * max(1, new))))
        return {"family": family, "model": model, "groups": groups, "batch": batch,
                "prefix_lo": rng.choice([0, prefix // 2, prefix]), "prefix_hi": prefix, "lo": rng.choice([0, 1]),
                "hi": _log(rng, 2, min(2000, 150000 // batch)), "new": new, "page": page, "lens": lens}
    if family == "window":
        new = rng.choice([0, 0, -1, _log(rng, 2, 700)])
        batch = _log(rng, 1, 256 if new == 0 else 8)
        hi = _log(rng, 40, min(30000, 2000000 // batch)) if new == 0 else _log(rng, 40, 10000 // batch)
        return {"family": family, "model": model, "batch": batch, "lo": rng.randint(1, hi), "hi": hi, "new": new,
                "window": _log(rng, 1, min(4000, 200000 // batch) if new == 0 else 1000) - 1,
                "first": _log(rng, 1, 200), "lse": rng.random() < 0.5, "page": page, "lens": lens}
    states = _log(rng, 1, 32)
    heads, dim = rng.choice([(32, 128), (32, 64), (64, 64), (16, 256), (8, 128), (14, 128)])
    tokens = _log(rng, 1, min(8192, 3000000 // (states * heads)))
    return {"family": family, "states": states, "tokens": tokens, "heads": heads, "dim": dim,
            "dtype": rng.choice(["bf16", "fp32"])}


# ------------------------------------------------------------------------------- batches
def _lens(case):
    """shared: (requests of each group, prefix lengths, suffix lengths, new tokens per request).
    window: (lengths, new tokens per request)."""
    r = random.Random(case["lens"])
    n = case["batch"]
    if case["family"] == "shared":
        cuts = sorted(r.randint(0, n) for _ in range(case["groups"] - 1))
        sizes = [b - a for a, b in zip([0] + cuts, cuts + [n])]
        prefix = [r.randint(case["prefix_lo"], case["prefix_hi"]) for _ in sizes]
        new = [r.randint(1, case["new"]) if case["new"] else 1 for _ in range(n)]
        # (a decode step's own token may be its suffix's only one; without it the suffix is empty)
        suffix = [r.randint(case["lo"], case["hi"]) + (k if case["new"] else 0) for k in new]
        return sizes, prefix, suffix, new
    total = [r.randint(case["lo"], case["hi"]) for _ in range(n)]
    if case["new"] == 0:
        return total, [1] * n
    return total, [t if case["new"] < 0 else min(t, r.randint(1, case["new"])) for t in total]


def _gen(seed, what):
    return torch.Generator(device="cuda").manual_seed(seed * 64 + what)


def _i32(xs):
    return torch.tensor(xs, dtype=torch.int32, device="cuda")


def _cum(xs):
    at = [0]
    for x in xs:
        at.append(at[-1] + x)
    return at


def _last(total, page):
    """Tokens on the last page of a run of `total` tokens."""
    return total - page * (-(-total // page) - 1) if total else 0


def _queries(shape, seed):
    """Query rows whose heads differ in sharpness, as a model's do."""
    sharp = torch.rand((1, shape[1], 1), generator=_gen(seed, 5), device="cuda") * 2 + 0.5
    return (torch.randn(shape, generator=_gen(seed, 6), device="cuda") * sharp).to(BF16)


def prepare(case, seed):
    s = {"case": case}
    if case["family"] == "merge":
        S, T, H, D = case["states"], case["tokens"], case["heads"], case["dim"]
        dtype = BF16 if case["dtype"] == "bf16" else torch.float32
        s["parts"] = torch.randn((S, T, H, D), generator=_gen(seed, 1), device="cuda", dtype=dtype)
        s["lses"] = torch.randn((S, T, H), generator=_gen(seed, 2), device="cuda") * 3 + 8
        blank = torch.rand((S, T, H), generator=_gen(seed, 3), device="cuda") < 0.05  # parts that saw nothing
        s["lses"].masked_fill_(blank, -math.inf)
        s["parts"].masked_fill_(blank[..., None], 0)
        return s
    Hq, Hkv, D = HEADS[case["model"]]
    P, shared = case["page"], case["family"] == "shared"
    if shared:
        sizes, prefix, suffix, new = _lens(case)
        runs = prefix + suffix  # runs of cached tokens: the groups', then the requests'
    else:
        runs, new = _lens(case)
    pages = [-(-t // P) for t in runs]
    pool = max(1, sum(pages))
    indptr = _cum(pages)
    indices = torch.randperm(pool, generator=_gen(seed, 4), device="cuda").to(torch.int32)
    s["q"] = _queries((sum(new), Hq, D), seed)
    s["cache"] = torch.randn((pool, 2, P, Hkv, D), generator=_gen(seed, 7), device="cuda", dtype=BF16)
    g = len(sizes) if shared else 0
    at = indptr[g]  # the requests' first page-table entry
    t = {"kv_indptr": _i32([x - at for x in indptr[g:]]), "kv_indices": indices[at:],
         "kv_last": _i32([_last(x, P) for x in runs[g:]]), "qo_indptr": _i32(_cum(new))}
    if shared:
        t.update(group_indptr=_i32(_cum(sizes)), prefix_indptr=_i32(indptr[:g + 1]), prefix_indices=indices[:at],
                 prefix_last=_i32([_last(x, P) for x in prefix]))
    s["tables"] = t
    if own:
        from pie_amd import attention

        ws = torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda")
        visible = {} if shared else {"window_left": case["window"], "first_tokens": case["first"]}
        kv = (t["kv_indptr"], t["kv_indices"], t["kv_last"])
        if shared:
            s["wrapper"] = attention.BatchSharedPrefixAttentionWrapper(ws, "NHD")
            s["wrapper"].plan(t["group_indptr"], t["prefix_indptr"], t["prefix_indices"], t["prefix_last"], *kv, Hq,
                              Hkv, D, P, qo_indptr=t["qo_indptr"] if case["new"] else None)
        elif case["new"] == 0:
            s["wrapper"] = attention.BatchDecodeWithPagedKVCacheWrapper(ws, "NHD")
            s["wrapper"].plan(*kv, Hq, Hkv, D, P, q_data_type=BF16, **visible)
        else:
            s["wrapper"] = attention.BatchPrefillWithPagedKVCacheWrapper(ws, "NHD")
            s["wrapper"].plan(t["qo_indptr"], *kv, Hq, Hkv, D, P, causal=True, q_data_type=BF16, **visible)
        return s
    # the plain form's plan: dense index tables
    s["kv"] = _dense(t["kv_indptr"], t["kv_indices"], runs[g:], P)
    rows = torch.arange(max(new), device="cuda")
    new_t, total = torch.tensor(new, device="cuda")[:, None], torch.tensor(runs[g:], device="cuda")[:, None]
    s["rows"] = (t["qo_indptr"][:-1, None] + torch.minimum(rows, new_t - 1)).long()  # [B, N] query token of each slot
    s["token"] = (rows < new_t).nonzero(as_tuple=True)  # and the (request, slot) of each token
    pos = total - new_t + rows  # position of each slot's token among its request's
    key = torch.arange(s["kv"][0].shape[1], device="cuda")
    if shared:
        # (a request without a suffix still decodes: it sees its prefix alone)
        s["see"] = ((key <= pos[..., None]) & (key < total[..., None]))[:, None, :, None, :]
        s["prefix"] = _dense(t["prefix_indptr"], t["prefix_indices"], prefix, P)
        first = [_cum(new)[b] for b in _cum(sizes)]
        count = torch.tensor([b - a for a, b in zip(first, first[1:])], device="cuda")[:, None]
        slot = torch.arange(max(1, int(count.max())), device="cuda")
        s["group_rows"] = (torch.tensor(first[:-1], device="cuda")[:, None] + slot).clamp(max=sum(new) - 1)
        s["group_token"] = (slot < count).nonzero(as_tuple=True)
        key = torch.arange(s["prefix"][0].shape[1], device="cuda")
        s["group_see"] = (key < torch.tensor(prefix, device="cuda")[:, None])[:, None, None, None, :]
    elif case["new"]:
        p = pos[..., None]
        s["see"] = ((key <= p) & ((key >= p - case["window"]) | (key < case["first"])))[:, None, :, None, :]
    else:
        # one query token each: only the positions it sees are gathered
        lo = (total - 1 - case["window"]).clamp(min=0)
        kept = lo.clamp(max=case["first"])
        j = torch.arange(int((kept + total - lo).max()), device="cuda")
        at = torch.where(j < kept, j, j - kept + lo).clamp(max=key.numel() - 1)
        s["kv"] = tuple(x.gather(1, at) for x in s["kv"])
        s["see"] = (j < kept + total - lo)[:, None, None, None, :]
    return s


def _dense(indptr, indices, lens, page):
    """(page, slot) of every position of every run, [runs, longest], padded with valid entries."""
    j = torch.arange(max(1, max(lens)), device="cuda")
    entry = (indptr[:-1, None].long() + j // page).clamp(max=max(0, indices.numel() - 1))
    if not indices.numel():
        return torch.zeros_like(entry), (j % page).expand_as(entry)
    return indices.long()[entry], (j % page).expand_as(entry)


# ------------------------------------------------------------------------------- one pass
def _part(q, cache, where, see, heads):
    """Attention of rows q [b, n, Hq, D] over the positions `where` [b, l], as (weighted value sums,
    softmax masses relative to the maxima, maxima of the base-2 scores): [b, n, Hq, D or 1]."""
    Hq, Hkv, D = heads
    b, n = q.shape[:2]
    q = q.float().view(b, n, Hkv, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(b, Hkv, -1, D)
    k = cache[where[0], 0, where[1]].float().permute(0, 2, 3, 1).contiguous()
    x = torch.matmul(q, k).mul_(LOG2E / math.sqrt(D)).view(b, Hkv, n, Hq // Hkv, -1)
    x = x.masked_fill_(~see, -math.inf)
    m = x.amax(-1, keepdim=True)
    x = torch.exp2(x.sub_(m.clamp(min=-1e30)))
    v = cache[where[0], 1, where[1]].float().transpose(1, 2).contiguous()
    o = torch.matmul(x.view(b, Hkv, -1, x.shape[-1]), v)
    back = lambda t: t.reshape(b, Hkv, n, Hq // Hkv, -1).transpose(1, 2).reshape(b, n, Hq, -1)
    return back(o), back(x.sum(-1)), back(m)


def run(state):
    s, case = state, state["case"]
    if case["family"] == "merge":
        if own:
            from pie_amd import attention

            out, lse = attention.merge_attention_states(s["parts"], s["lses"])
            return {"out": out, "lse": lse}
        m = s["lses"].amax(0)
        w = torch.exp2(s["lses"] - m.clamp(min=-1e30))
        total = w.sum(0)
        out = (w[..., None] * s["parts"].float()).sum(0) / total.clamp(min=1e-30)[..., None]
        return {"out": out.to(s["parts"].dtype), "lse": m + torch.log2(total)}
    with_lse = case.get("lse", False)
    if own:
        if with_lse:
            out, lse = s["wrapper"].run(s["q"], s["cache"], return_lse=True)
            return {"out": out, "lse": lse}
        return {"out": s["wrapper"].run(s["q"], s["cache"])}
    heads, q = HEADS[case["model"]], s["q"]
    o, l, m = (x[s["token"]] for x in _part(q[s["rows"]], s["cache"], s["kv"], s["see"], heads))
    if case["family"] == "shared":
        po, pl, pm = (x[s["group_token"]] for x in _part(q[s["group_rows"]], s["cache"], s["prefix"], s["group_see"], heads))
        top = torch.maximum(m, pm)
        ref = top.clamp(min=-1e30)
        a, b = torch.exp2(m - ref), torch.exp2(pm - ref)
        o, l, m = o * a + po * b, l * a + pl * b, top
    result = {"out": (o / l.clamp(min=1e-30)).to(BF16)}
    if with_lse:
        result["lse"] = (m + torch.log2(l))[..., 0]
    return result


# ------------------------------------------------------------------------------- work
def work(case):
    if case["family"] == "merge":
        rows, size = case["tokens"] * case["heads"], 2 if case["dtype"] == "bf16" else 4
        each = rows * (case["dim"] * size + 4)
        return {"bytes": (case["states"] + 1) * each, "flops": 2 * case["states"] * rows * case["dim"]}
    Hq, Hkv, D = HEADS[case["model"]]
    P = case["page"]
    pairs = seen = 0
    if case["family"] == "shared":
        sizes, prefix, suffix, new = _lens(case)
        first = _cum(sizes)
        for g, length in enumerate(prefix):
            tokens = sum(new[first[g]:first[g + 1]])
            pairs += tokens * length
            seen += length if tokens else 0
        for total, n in zip(suffix, new):
            pairs += sum(max(0, total - n + i + 1) for i in range(n)) if case["new"] else total
            seen += total
        T, tables = sum(new), len(prefix) + len(suffix)
    else:
        total, new = _lens(case)
        W, F = case["window"], case["first"]
        for t, n in zip(total, new):
            pairs += sum(min(p + 1, W + 1 + min(F, max(0, p - W))) for p in range(t - n, t))
            lo = max(0, t - n - W)
            seen += t - lo + min(F, lo)
        T, tables = sum(new), len(total)
    size = 4 * T * Hq * D + 4 * seen * Hkv * D + 4 * (seen // P) + 12 * tables
    return {"bytes": size + (4 * T * Hq if case.get("lse") else 0), "flops": 4 * pairs * Hq * D}


# ------------------------------------------------------------------------------- 64-bit results
def exact(case, seed):
    s = prepare(case, seed)
    if case["family"] == "merge":
        lses, parts = s["lses"].double(), s["parts"].double()
        lse = torch.logsumexp(lses * math.log(2), 0) / math.log(2)
        share = torch.nan_to_num(torch.softmax(lses * math.log(2), 0))  # (0 where no part saw anything)
        return {"out": (share[..., None] * parts).sum(0), "lse": lse}
    Hq, Hkv, D = HEADS[case["model"]]
    t, G, P, shared = s["tables"], Hq // Hkv, case["page"], case["family"] == "shared"

    def tokens(indptr, indices, i, length):
        """k and v of run i, [Hkv, length, D] in 64 bits."""
        page = indices[int(indptr[i]):int(indptr[i + 1])].long()
        kv = s["cache"][page].transpose(1, 2).reshape(-1, 2, Hkv, D)[:length].double()
        return kv[:, 0].transpose(0, 1).contiguous(), kv[:, 1].transpose(0, 1).contiguous()

    if shared:
        sizes, prefix, suffix, new = _lens(case)
        group = [g for g, n in enumerate(sizes) for _ in range(n)]
        runs = suffix
    else:
        runs, new = _lens(case)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    at, held = 0, (None, None)
    for b, (length, n) in enumerate(zip(runs, new)):
        k, v = tokens(t["kv_indptr"], t["kv_indices"], b, length)
        ahead = 0
        if shared:
            if held[0] != group[b]:
                held = (group[b], tokens(t["prefix_indptr"], t["prefix_indices"], group[b], prefix[group[b]]))
            ahead = prefix[group[b]]
            k, v = torch.cat([held[1][0], k], 1), torch.cat([held[1][1], v], 1)
        # the queries are the last n positions (a request without a suffix asks from behind its prefix)
        p = torch.arange(n, device="cuda")[:, None] + ahead + length - n
        j = torch.arange(ahead + length, device="cuda")[None, :]
        hidden = j > p.clamp(min=ahead - 1)
        if not shared:
            hidden = hidden | ((j < p - case["window"]) & (j >= case["first"]))
        if k.shape[1]:
            for h in range(Hq):
                x = s["q"][at:at + n, h].double() @ k[h // G].t().contiguous() / math.sqrt(D)
                x = x.masked_fill(hidden, -math.inf)
                out[at:at + n, h] = torch.nan_to_num(torch.softmax(x, -1)) @ v[h // G]
                lse[at:at + n, h] = torch.logsumexp(x, -1) / math.log(2)
        at += n
    return {"out": out, "lse": lse} if case.get("lse") else {"out": out}
