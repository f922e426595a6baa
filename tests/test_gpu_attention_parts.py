"""GPU: attention over parts of a paged cache against plain float64 torch: first tokens kept visible
beside a window (decode and prefill), log-sum-exps, prefixes shared by groups of requests, and the join of
results over parts.

Tolerance of a bf16 output row, with A = sum_t p_t |v_t| of that element: the probabilities enter the
second product rounded to bf16 and the output is rounded once, each off by at most half a step (2^-8
relative): 2^-8 (A + |o|). A score's fp32 sum of D <= 256 products is off by at most D 2^-24 sum|q_d k_d|
scale log2(e) < 2^-11 for N(0, 1) data, which the probabilities take over relatively: 2^-11 A, and with
it the log-sum-exp absolutely; the sums over up to 2^15 positions in fp32 stay far below both."""
from __future__ import annotations

import math

import pytest
import torch

from pie_amd import _lib, attention

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(xs, dev):
    return torch.tensor(list(xs), dtype=torch.int32, device=dev)


def _cum(xs):
    at = [0]
    for x in xs:
        at.append(at[-1] + x)
    return at


def _ws(dev, size=64 << 20):
    return torch.zeros(size, dtype=torch.uint8, device=dev)


class Cache:
    """A paged cache of N(0, 1) values whose pages are handed out in random order as runs of tokens."""

    def __init__(self, dev, pages, P, Hkv, D, layout="NHD", split=False, seed=0):
        shape = (pages, 2, P, Hkv, D) if layout == "NHD" else (pages, 2, Hkv, P, D)
        self.data = torch.randn(shape, generator=_gen(seed), device=dev, dtype=BF16)
        self.arg = (self.data[:, 0], self.data[:, 1]) if split else self.data
        self.order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.P, self.layout, self.dev, self.used = P, layout, dev, 0

    def runs(self, lens):
        """(indptr, indices, last_page_len) tables of runs of these lengths, and their page ids."""
        pages = [-(-n // self.P) for n in lens]
        ids = [self.order[self.used + a:self.used + b] for a, b in zip(_cum(pages), _cum(pages)[1:])]
        self.used += sum(pages)
        last = [n - self.P * (p - 1) if p else 0 for n, p in zip(lens, pages)]
        return (_i32(_cum(pages), self.dev), _i32([i for x in ids for i in x], self.dev), _i32(last, self.dev)), ids

    def tokens(self, ids, length):
        """k and v of a run, [length, Hkv, D]."""
        kv = self.data[torch.tensor(ids, dtype=torch.long, device=self.dev)]
        if self.layout == "HND":
            kv = kv.transpose(2, 3)
        kv = kv.transpose(1, 2).reshape(-1, 2, kv.shape[3], kv.shape[4])[:length]
        return kv[:, 0], kv[:, 1]


def _plain(q, k, v, see, scale=None):
    """float64 (out, A = sum p|v|, base-2 lse) of rows q [n, Hq, D] over k, v [l, Hkv, D]; see [n, l]."""
    n, Hq, D = q.shape
    G = Hq // k.shape[1] if k.shape[1] else 1
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    A, lse = out.clone(), torch.full((n, Hq), -math.inf, dtype=torch.float64, device=q.device)
    if k.shape[0] == 0:
        return out, A, lse
    for h in range(Hq):
        s = q[:, h].double() @ k[:, h // G].double().t().contiguous() * (D ** -0.5 if scale is None else scale)
        s = s.masked_fill(~see, -math.inf)
        p = torch.nan_to_num(torch.softmax(s, -1)).masked_fill(~see, 0)
        vh = torch.where(see.any(0)[:, None], v[:, h // G].double(), 0.0)  # (nobody's positions may hold NaN)
        out[:, h], A[:, h] = p @ vh, p @ vh.abs()
        lse[:, h] = torch.logsumexp(s, -1) / math.log(2)
    return out, A, lse


def _compare(got, want, what):
    """got: out or (out, lse); want: _plain's."""
    out, A, lse = want
    g = got[0] if isinstance(got, tuple) else got
    off = (g.double() - out).abs() / (2 ** -8 * (A + out.abs()) + 2 ** -11 * A + 1e-30)
    assert not torch.isnan(g).any(), f"{what}: NaN"
    assert off.numel() == 0 or off.max() <= 1, f"{what}: {off.max().item():.3f} of the tolerance"
    if isinstance(got, tuple):
        e = got[1].double()
        assert torch.equal(torch.isinf(e), torch.isinf(lse)), f"{what}: which rows see nothing"
        fin = torch.isfinite(lse)
        far = (e[fin] - lse[fin]).abs() / (2 ** -11 + 2 ** -20 * lse[fin].abs())
        assert far.numel() == 0 or far.max() <= 1, f"{what}: lse {far.max().item():.3f} of the tolerance"


def _cat(parts):
    return tuple(torch.cat(x) for x in zip(*parts))


# ----------------------------------------------------------------- windows that keep first tokens
def _window_case(dev, lens, news, heads, P, window, first, mode=1, layout="NHD", split=False, seed=1, masks=None,
                 poison=False):
    Hq, Hkv, D = heads
    c = Cache(dev, max(1, sum(-(-n // P) for n in lens)), P, Hkv, D, layout, split, seed)
    tables, ids = c.runs(lens)
    T = sum(news)
    qkv = torch.randn((T, (Hq + 2 * Hkv) * D), generator=_gen(seed + 1), device=dev, dtype=BF16)
    q = qkv[:, :Hq * D].view(T, Hq, D)  # a strided view, as the projections give
    want, at = [], 0
    for b, (n, new) in enumerate(zip(lens, news)):
        p = torch.arange(new, device=dev)[:, None] + n - new
        t = torch.arange(n, device=dev)[None]
        see = masks[b] if mode == 2 else (t <= p if mode == 1 else torch.ones((new, n), dtype=torch.bool, device=dev))
        if window >= 0:
            see = see & ((t >= p - window) | (t < first))
        if poison and new:  # positions before every window and past the first tokens hold NaN
            for j in range(min(first, n), max(0, n - new - window)):
                (c.data[ids[b][j // P], :, j % P] if layout == "NHD" else c.data[ids[b][j // P], :, :, j % P]).fill_(math.nan)
        k, v = c.tokens(ids[b], n)
        want.append(_plain(q[at:at + new], k, v, see))
        at += new
    return c, tables, q, _cat(want)


HEADS = [(32, 8, 128), (14, 2, 64), (16, 8, 256), (8, 8, 128), (16, 1, 64)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("P,layout,split", [(16, "NHD", False), (5, "HND", False), (1, "NHD", True)])
@pytest.mark.parametrize("window,first", [(0, 1), (63, 4), (100, 33), (700, 600), (5000, 3), (-1, 9), (0, 0)])
def test_decode_window_with_first_tokens(dev, heads, P, layout, split, window, first):
    lens = [1, 40, 64, 0, 65, 333, 1500]
    print(f"decode {heads} P={P} {layout} window={window} first={first}", flush=True)
    c, (ip, ix, ll), q, want = _window_case(dev, lens, [1] * len(lens), heads, P, window, first, layout=layout, split=split)
    w = attention.BatchDecodeWithPagedKVCacheWrapper(_ws(dev), layout)
    for tables in ((ip, ix, ll), (ip.cpu(), ix.cpu(), ll.cpu())):
        w.plan(*tables, *heads, P, q_data_type=BF16, window_left=window, first_tokens=first)
        _compare(w.run(q, c.arg, return_lse=True), want, "decode")
    assert torch.equal(w.run(q, c.arg), w.run(q, c.arg, return_lse=True)[0])


@pytest.mark.parametrize("batch", [1, 3, 300])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_lse_at_any_split(dev, batch, D):
    """One split writes its log-sum-exps itself, several in the merge; batches past 256 keep request order."""
    heads = (8, 2, D)
    lens = [(37 * b) % 700 for b in range(batch)]
    c, tables, q, want = _window_case(dev, lens, [1] * batch, heads, 16, 127, 4, seed=5)
    w = attention.BatchDecodeWithPagedKVCacheWrapper(_ws(dev, batch * 64 * 8 * (D + 1) * 4 + (1 << 20)), "NHD")
    w.plan(*tables, *heads, 16, q_data_type=BF16, window_left=127, first_tokens=4)
    for splits in (1, 2, 5, 64):
        w._plan["splits"] = splits
        _compare(w.run(q, c.arg, return_lse=True), want, f"splits {splits}")


PREFILLS = [
    ([300, 40, 0, 1], [60, 40, 0, 1], 63, 4),   # chunks and a whole prompt, an empty request
    ([1000], [1000], 100, 5),                   # one prompt many windows long
    ([900, 2000], [13, 3], 500, 200),           # a few tokens over long contexts (cut over kv)
    ([5000], [9], 4000, 130),                   # pieces on both sides of the seam
    ([5000], [9], 300, 4000),                   # first tokens most of the context
    ([200], [40], 0, 1),
    ([130, 70], [130, 70], -1, 9),              # no window: first tokens change nothing
]


@pytest.mark.parametrize("heads", [(32, 8, 128), (14, 2, 64), (16, 8, 256), (4, 4, 128)])
@pytest.mark.parametrize("lens,news,window,first", PREFILLS)
def test_prefill_window_with_first_tokens(dev, heads, lens, news, window, first):
    for P, layout, split in ((16, "NHD", False), (5, "HND", True)):
        print(f"prefill {heads} {lens} window={window} first={first} P={P}", flush=True)
        c, tables, q, want = _window_case(dev, lens, news, heads, P, window, first, layout=layout, split=split)
        w = attention.BatchPrefillWithPagedKVCacheWrapper(_ws(dev), layout)
        w.plan(_i32(_cum(news), dev), *tables, *heads, P, causal=True, q_data_type=BF16, window_left=window,
               first_tokens=first)
        _compare(w.run(q, c.arg, return_lse=True), want, "prefill")
        assert torch.equal(w.run(q, c.arg), w.run(q, c.arg, return_lse=True)[0])


@pytest.mark.parametrize("mode", [0, 2])
@pytest.mark.parametrize("heads", [(8, 2, 128), (8, 2, 64), (4, 2, 256)])
def test_prefill_first_tokens_in_other_modes(dev, heads, mode):
    lens, news = [400, 90, 1600], [50, 90, 7]
    g = torch.Generator().manual_seed(3)
    masks = [(torch.rand((n, t), generator=g) < 0.6).to(dev) for t, n in zip(lens, news)]
    masks[0][5] = False  # a row whose mask leaves nothing
    c, tables, q, want = _window_case(dev, lens, news, heads, 16, 77, 20, mode=mode, masks=masks)
    w = attention.BatchPrefillWithPagedKVCacheWrapper(_ws(dev), "NHD")
    kw = {"custom_mask": torch.cat([m.flatten() for m in masks])} if mode == 2 else {}
    w.plan(_i32(_cum(news), dev), *tables, *heads, 16, q_data_type=BF16, window_left=77, first_tokens=20, **kw)
    _compare(w.run(q, c.arg, return_lse=True), want, f"mode {mode}")


def test_prefill_lse_on_many_work_items(dev):
    """More units than the chip runs at once: the persistent kernel's log-sum-exps (head dim 128)."""
    heads, lens = (32, 8, 128), [200 + b for b in range(40)]
    c, tables, q, want = _window_case(dev, lens, lens, heads, 16, -1, 0)
    w = attention.BatchPrefillWithPagedKVCacheWrapper(_ws(dev), "NHD")
    w.plan(_i32(_cum(lens), dev), *tables, *heads, 16, causal=True, q_data_type=BF16)
    _compare(w.run(q, c.arg, return_lse=True), want, "prefill")


@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_hidden_positions_are_not_seen(dev, new, D):
    """What lies between the first tokens and every window: NaN keys and values, then page ids outside
    the pool, as a stream whose passed pages were given away leaves them."""
    heads, window, first, lens = (8, 2, D), 90, 7, [1000, 700, 150]
    c, (ip, ix, ll), q, want = _window_case(dev, lens, [new] * 3, heads, 16, window, first, poison=True)

    def run(ix):
        if new == 1:
            w = attention.BatchDecodeWithPagedKVCacheWrapper(_ws(dev), "NHD")
            w.plan(ip, ix, ll, *heads, 16, q_data_type=BF16, window_left=window, first_tokens=first)
        else:
            w = attention.BatchPrefillWithPagedKVCacheWrapper(_ws(dev), "NHD")
            w.plan(_i32(_cum([new] * 3), dev), ip, ix, ll, *heads, 16, causal=True, q_data_type=BF16, window_left=window,
                   first_tokens=first)
        return w.run(q, c.arg, return_lse=True)

    _compare(run(ix), want, "NaN between")
    gone = ix.clone()
    at = ip.tolist()
    for b, n in enumerate(lens):
        gone[at[b] + 1:at[b] + max(1, (n - new - window) // 16)] = 2 ** 30  # pages of hidden positions only
    _compare(run(gone), want, "pages given away")


def test_sink_attention_with_first_tokens(dev):
    heads, window, first = (64, 8, 64), 127, 4
    Hq = heads[0]
    sinks = torch.randn(Hq, generator=_gen(9), device=dev)
    for lens, news in (([400, 90, 1], [1, 1, 1]), ([400, 90], [30, 90])):
        c, tables, q, (out, A, lse) = _window_case(dev, lens, news, heads, 16, window, first)
        w = attention.BatchAttentionWithAttentionSinkWrapper(_ws(dev), "NHD", window_left=window)
        w.plan(_i32(_cum(news), dev), *tables, *heads, 16, first_tokens=first)
        part = 1 / (1 + torch.exp2(sinks.double() * math.log2(math.e) - lse))[..., None]  # the positions' share
        _compare(w.run(q, c.arg, sinks), (out * part, A * part, lse), "sinks")
        with pytest.raises(NotImplementedError):
            w.run(q, c.arg, sinks, return_lse=True)


def test_captured_decode_window_follows_its_tables(dev):
    """A captured run with first tokens, replayed over tables that grow past the window."""
    heads, P, window, first = (8, 2, 128), 16, 60, 5
    c = Cache(dev, 64, P, *heads[1:], seed=3)
    c.order = list(range(64))
    ip, ix, ll = _i32([0, 32, 64], dev), _i32(range(64), dev), _i32([0, 0], dev)
    fixed = (torch.zeros(3, dtype=torch.int32, device=dev), ix.clone(), torch.zeros(2, dtype=torch.int32, device=dev))
    w = attention.BatchDecodeWithPagedKVCacheWrapper(_ws(dev), "NHD", use_cuda_graph=True, paged_kv_indptr_buffer=fixed[0],
                                                     paged_kv_indices_buffer=fixed[1], paged_kv_last_page_len_buffer=fixed[2])
    q = torch.randn((2, 8, 128), generator=_gen(4), device=dev, dtype=BF16)
    out, lse = torch.empty_like(q), torch.empty((2, 8), device=dev)

    def tables(lens):
        pages = [-(-n // P) for n in lens]
        flat = [i for b, p in enumerate(pages) for i in range(32 * b, 32 * b + p)]
        return _i32(_cum(pages), dev), _i32(flat + [0] * (64 - len(flat)), dev), _i32([n - P * (p - 1) for n, p in zip(lens, pages)], dev)

    w.plan(*tables([3, 70]), *heads, P, q_data_type=BF16, window_left=window, first_tokens=first)
    w.run(q, c.arg, out=out, lse=lse)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w.run(q, c.arg, out=out, lse=lse)
    for lens in ([3, 70], [65, 66], [500, 62], [511, 512]):
        for b, t in zip(fixed, tables(lens)):
            b.copy_(t)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        want = []
        for b, n in enumerate(lens):
            k, v = c.tokens(list(range(32 * b, 32 * b + 32)), n)
            t = torch.arange(n, device=dev)[None]
            want.append(_plain(q[b:b + 1], k, v, (t >= n - 1 - window) | (t < first)))
        _compare((out, lse), _cat(want), f"replay {lens}")


# ----------------------------------------------------------------------------- shared prefixes
def _shared_case(dev, sizes, prefixes, suffixes, news, heads, P, layout="NHD", split=False, seed=1):
    """news None: one query token per request."""
    Hq, Hkv, D = heads
    pages = sum(-(-n // P) for n in prefixes + suffixes)
    c = Cache(dev, max(1, pages), P, Hkv, D, layout, split, seed)
    pre, pre_ids = c.runs(prefixes)
    suf, suf_ids = c.runs(suffixes)
    T = sum(news) if news else len(suffixes)
    q = torch.randn((T, (Hq + 2 * Hkv) * D), generator=_gen(seed + 1), device=dev, dtype=BF16)[:, :Hq * D].view(T, Hq, D)
    group = [g for g, n in enumerate(sizes) for _ in range(n)]
    want, at = [], 0
    for b, n in enumerate(suffixes):
        m, g = news[b] if news else 1, group[b]
        (pk, pv), (sk, sv) = c.tokens(pre_ids[g], prefixes[g]), c.tokens(suf_ids[b], n)
        t, i = torch.arange(prefixes[g] + n, device=dev)[None], torch.arange(m, device=dev)[:, None]
        see = (t < prefixes[g]) | (t <= prefixes[g] + n - m + i) | (torch.tensor(not news, device=dev))
        want.append(_plain(q[at:at + m], torch.cat([pk, sk]), torch.cat([pv, sv]), see))
        at += m
    args = (_i32(_cum(sizes), dev), *pre, *suf)
    kw = {"qo_indptr": _i32(_cum(news), dev)} if news else {}
    return c, args, kw, q, _cat(want)


SHARED = [
    ([4], [600], [1, 33, 0, 60], None),
    ([3, 0, 2, 1], [70, 500, 0, 129], [5, 0, 90, 300, 1, 0], None),   # empty group, prefix and suffixes
    ([2, 1], [0, 0], [0, 0, 7], None),                                # rows that see nothing
    ([1] * 7, [1, 15, 16, 17, 255, 256, 257], [1] * 7, None),         # nothing shared
    ([40], [5000], [1 + 40 * b for b in range(40)], None),            # many rows, long and unequal suffixes
    ([270], [100], [b % 5 for b in range(270)], None),                # past 256 requests
    ([1], [20000], [2000], None),
    ([3, 2], [150, 40], [9, 30, 4, 12, 60], [9, 5, 1, 0, 3]),
    ([2, 1, 3], [2000, 0, 31], [700, 300, 1, 40, 40, 200], [40, 2, 1, 33, 40, 13]),
    ([1], [64], [3], [5]),                                            # more query tokens than the suffix holds
]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("sizes,prefixes,suffixes,news", SHARED)
def test_shared_prefix(dev, heads, sizes, prefixes, suffixes, news):
    for P, layout, split in ((16, "NHD", False), (5, "HND", False), (1, "NHD", True)):
        print(f"shared {heads} {sizes} {prefixes} P={P} {layout}", flush=True)
        c, args, kw, q, want = _shared_case(dev, sizes, prefixes, suffixes, news, heads, P, layout, split)
        w = attention.BatchSharedPrefixAttentionWrapper(_ws(dev), layout)
        w.plan(*args, *heads, P, **kw)
        _compare(w.run(q, c.arg, return_lse=True), want, "shared")
        w.plan(*(t.cpu() for t in args), *heads, P, **{k: v.cpu() for k, v in kw.items()})
        out = torch.full((q.shape[0] + 2, *q.shape[1:]), 7.0, dtype=BF16, device=dev)
        lse = torch.full((q.shape[0] + 2, q.shape[1]), 7.0, device=dev)
        got = w.run(q, c.arg, out=out[1:-1], lse=lse[1:-1])
        assert got.data_ptr() == out[1:-1].data_ptr()
        _compare((got, lse[1:-1]), want, "shared, tables on the host")
        for t in (out, lse):  # rows before the first token and behind the last
            assert (t[0] == 7).all() and (t[-1] == 7).all()


JOINT = [  # (sizes, prefixes, suffixes, news, joined: some group's parts are joined)
    ([3, 0, 2, 1], [500, 9, 0, 65], [40, 7, 64, 3, 1, 90], [40, 1, 33, 3, 1, 20], False),
    ([1, 1], [64, 1], [5, 200], [9, 150], False),           # more query tokens than the suffix holds, many rows
    ([2, 2, 1], [3000, 200, 400], [30, 2, 70, 5, 9], [13, 2, 5, 5, 9], True),
    ([1, 2], [100, 30], [3000, 4, 8], [7, 4, 1], True),     # a suffix in pieces: its group is joined
]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("sizes,prefixes,suffixes,news,joined", JOINT)
def test_short_prefixes_with_several_query_tokens(dev, heads, sizes, prefixes, suffixes, news, joined):
    """Items that walk a prefix and their suffix and write the output, alone and beside parts that are joined; NaN in
    the slots behind a run's last token; replays of a captured run between eager ones."""
    for P, layout in ((16, "NHD"), (5, "HND"), (1, "NHD")):
        print(f"short prefixes {heads} {prefixes} P={P} {layout}", flush=True)
        c, args, kw, q, want = _shared_case(dev, sizes, prefixes, suffixes, news, heads, P, layout)
        for ip, ix, ll in (args[1:4], args[4:7]):
            for i, (a, b, n) in enumerate(zip(ip.tolist(), ip.tolist()[1:], ll.tolist())):
                if b > a:
                    page = c.data[ix[b - 1]]
                    (page[:, n:] if layout == "NHD" else page[:, :, n:]).fill_(math.nan)
        whole = not joined and (heads[2] != 256 or max(prefixes) <= 128)
        w = attention.BatchSharedPrefixAttentionWrapper(_ws(dev, 64 if whole else 64 << 20), layout)
        w.plan(*args, *heads, P, **kw)
        assert (w._plan["info"][1] == 0) == whole
        out = torch.full((q.shape[0] + 2, *q.shape[1:]), 7.0, dtype=BF16, device=dev)
        lse = torch.full((q.shape[0] + 2, q.shape[1]), 7.0, device=dev)
        w.run(q, c.arg, out=out[1:-1], lse=lse[1:-1])
        _compare((out[1:-1], lse[1:-1]), want, "short prefixes")
        for t in (out, lse):
            assert (t[0] == 7).all() and (t[-1] == 7).all()
        if P == 16:
            eager = out.clone()
            g = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(g):
                w.run(q, c.arg, out=out[1:-1])
            for _ in range(3):
                out[1:-1].zero_()
                g.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, eager)
                w.run(q, c.arg)


def test_more_query_heads_per_kv_head_than_a_decode_tile(dev):
    c, args, kw, q, want = _shared_case(dev, [2], [300], [20, 9], [20, 3], (40, 2, 128), 16)
    w = attention.BatchSharedPrefixAttentionWrapper(_ws(dev))
    w.plan(*args, 40, 2, 128, 16, **kw)
    _compare(w.run(q, c.arg, return_lse=True), want, "20 heads per kv head")


def test_shared_prefix_in_little_workspace(dev):
    """Less workspace than the pieces want: longer pieces, same result; less than one piece each: refused."""
    heads = (8, 2, 128)
    c, args, kw, q, want = _shared_case(dev, [6], [9000], [400] * 6, None, heads, 16)
    w = attention.BatchSharedPrefixAttentionWrapper(_ws(dev))
    w.plan(*args, *heads, 16)
    full = w._plan["info"][1]
    small = attention.BatchSharedPrefixAttentionWrapper(_ws(dev, full // 4)[4:])  # (off a 16-byte boundary)
    small.plan(*args, *heads, 16)
    assert small._plan["info"][1] <= full // 4 - 16
    for x in (w, small):
        _compare(x.run(q, c.arg, return_lse=True), want, "little workspace")
    with pytest.raises(ValueError, match="workspace"):
        attention.BatchSharedPrefixAttentionWrapper(_ws(dev, 4096)).plan(*args, *heads, 16)


def test_shared_pages_outside_the_pool_are_masked(dev):
    heads = (8, 2, 128)
    c, args, kw, q, _ = _shared_case(dev, [3], [320], [40, 2, 100], None, heads, 16)
    args[2][3] = -1
    args[2][7] = 10 ** 6
    w = attention.BatchSharedPrefixAttentionWrapper(_ws(dev))
    w.plan(*args, *heads, 16)
    got = w.run(q, c.arg, return_lse=True)
    want = []
    at = args[4].tolist()
    for b, n in enumerate([40, 2, 100]):
        pk, pv = c.tokens([max(0, i) % 10 ** 6 for i in args[2].tolist()], 320)
        sk, sv = c.tokens(args[5].tolist()[at[b]:at[b + 1]], n)
        see = torch.ones((1, 320 + n), dtype=torch.bool, device=dev)
        see[:, 48:64] = see[:, 112:128] = False
        want.append(_plain(q[b:b + 1], torch.cat([pk, sk]), torch.cat([pv, sv]), see))
    _compare(got, _cat(want), "masked pages")


def test_one_captured_shared_run_follows_its_tables(dev):
    """Planned once: the captured run serves suffixes that grow and shrink, between eager runs of its own
    wrapper and others, and outlives a new plan of the wrapper."""
    heads, P, B = (32, 8, 128), 16, 6
    Hq, Hkv, D = heads
    c = Cache(dev, 40 + 32 * B, P, Hkv, D, seed=5)
    pre, pre_ids = c.runs([500, 77])
    room = [c.order[c.used + 32 * b:c.used + 32 * b + 32] for b in range(B)]
    ip, ix, ll = (torch.zeros(n, dtype=torch.int32, device=dev) for n in (B + 1, 32 * B, B))
    ws = _ws(dev)
    w = attention.BatchSharedPrefixAttentionWrapper(ws)
    q = torch.randn((B, Hq, D), generator=_gen(6), device=dev, dtype=BF16)
    out, lse = torch.empty_like(q), torch.empty((B, Hq), device=dev)

    def put(lens):
        pages = [-(-n // P) for n in lens]
        flat = [i for r, p in zip(room, pages) for i in r[:p]]
        ip.copy_(_i32(_cum(pages), dev))
        ix.copy_(_i32(flat + [0] * (32 * B - len(flat)), dev))
        ll.copy_(_i32([n - P * (p - 1) if p else 0 for n, p in zip(lens, pages)], dev))
        want = []
        for b, n in enumerate(lens):
            g = 0 if b < 4 else 1
            (pk, pv), (sk, sv) = c.tokens(pre_ids[g], [500, 77][g]), c.tokens(room[b], n)
            k = torch.cat([pk, sk])
            want.append(_plain(q[b:b + 1], k, torch.cat([pv, sv]), torch.ones((1, k.shape[0]), dtype=torch.bool, device=dev)))
        return _cat(want)

    args = (_i32([0, 4, 6], dev), *pre, ip, ix, ll, *heads, P)
    want = put([1] * B)
    w.plan(*args)
    _compare(w.run(q, c.arg, out=out, return_lse=True), want, "eager")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w.run(q, c.arg, out=out, lse=lse)
    for i, lens in enumerate(([1] * B, [0, 5, 16, 17, 300, 2], [512] * B, [3, 0, 0, 0, 0, 511])):
        want = put(lens)
        for _ in range(2):
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            _compare((out, lse), want, f"replay {lens}")
            _compare(w.run(q, c.arg, return_lse=True), want, f"eager {lens}")
        if i == 1:
            w.plan(*args)  # the graph keeps its own plan
            w.run(q, c.arg)


def test_shared_run_on_a_busy_workspace_is_refused(dev):
    heads = (32, 8, 128)
    c, args, kw, q, want = _shared_case(dev, [64], [16000], [1] * 64, None, heads, 16)
    w = attention.BatchSharedPrefixAttentionWrapper(_ws(dev))
    w.plan(*args, *heads, 16)
    outs = [torch.empty((64, 32, 128), dtype=BF16, device=dev) for _ in range(2)]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):  # (a stream's first use takes some ms)
        with torch.cuda.stream(s):
            torch.zeros(1, device=dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        for _ in range(40):  # ~1 ms queued on s1
            w.run(q, c.arg, out=outs[0])
    with torch.cuda.stream(s2):
        with pytest.raises(_lib.PieHipError, match="another stream"):
            w.run(q, c.arg, out=outs[1])
    s1.synchronize()
    with torch.cuda.stream(s2):
        w.run(q, c.arg, out=outs[1])
    torch.cuda.synchronize()
    assert torch.equal(*outs)
    _compare(outs[1], want, "second stream")


@pytest.mark.parametrize("heads", [(32, 8, 128), (6, 3, 64), (8, 4, 256)])
def test_many_requests(dev, heads):
    """More stream units than the device runs at once: two kv heads to a work group, where their number is even;
    suffixes of every length around the tiles' and pieces' ends."""
    suffixes = [(37 * b) % 300 for b in range(190)]
    c, args, kw, q, want = _shared_case(dev, [150, 3, 37], [700, 40, 129], suffixes, None, heads, 16)
    w = attention.BatchSharedPrefixAttentionWrapper(_ws(dev, 256 << 20))
    w.plan(*args, *heads, 16)
    got = w.run(q, c.arg, return_lse=True)
    _compare(got, want, "many requests")
    again = w.run(q, c.arg, return_lse=True)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("news", [None, [9, 1, 30, 4]])
def test_shared_prefix_at_other_scales(dev, news):
    heads = (32, 8, 128)
    c, args, kw, q, want = _shared_case(dev, [3, 1], [200, 33], [40, 9, 70, 4], news, heads, 16)
    w = attention.BatchSharedPrefixAttentionWrapper(_ws(dev))
    w.plan(*args, *heads, 16, sm_scale=-128 ** -0.5, **kw)
    _compare(w.run(-q, c.arg, return_lse=True), want, "a negative scale")
    w.plan(*args, *heads, 16, sm_scale=0.0, **kw)
    got = w.run(q, c.arg, return_lse=True)
    w.plan(*args, *heads, 16, **kw)
    mean = w.run(torch.zeros_like(q), c.arg, return_lse=True)
    assert torch.equal(got[0], mean[0]) and torch.allclose(got[1], mean[1], rtol=2 ** -22, atol=0)


def test_a_plan_outlives_runs_on_other_streams(dev):
    """A run queued on another stream than its plan's, then a new plan: the first one's memory is not handed
    out before the run has read it."""
    heads = (8, 2, 128)
    c, args, kw, q, want = _shared_case(dev, [40], [900], [3 + b for b in range(40)], None, heads, 16)
    w = attention.BatchSharedPrefixAttentionWrapper(_ws(dev))
    w.plan(*(t.cpu() for t in args), *heads, 16)
    made = [(t.numel(), t.data_ptr()) for t in w._plan["made"]]
    out, lse = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty(q.shape[:2], device=dev)
    s = torch.cuda.Stream()
    w.run(q, c.arg)  # (the kernels are loaded)
    big = torch.zeros(1 << 28, device=dev)
    with torch.cuda.stream(s):
        big.add_(1)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(200):  # ~100 ms before the run
            big.add_(1)
        w.run(q, c.arg, out=out, lse=lse)
    w.plan(*(t.cpu() for t in args), *heads, 16)
    new = [torch.full((n,), -1, dtype=torch.int32, device=dev) for n, _ in made for _ in range(4)]
    if not s.query():  # (the run was still queued: it is the memory of a run that has ended that may be handed out)
        assert not {t.data_ptr() for t in new + w._plan["made"]} & {at for _, at in made}
    torch.cuda.synchronize()
    _compare((out, lse), want, "another stream")


def test_offsets_past_32_bits(dev):
    """Pages whose elements lie past 2^32 bytes and 2^31 elements of the pool."""
    heads, P = (8, 4, 128), 32
    Hq, Hkv, D = heads
    pages = 2 ** 31 // (2 * P * Hkv * D) + 40
    data = torch.empty((pages, 2, P, Hkv, D), dtype=BF16, device=dev)
    ids = list(range(pages - 24, pages)) + [0, 1]
    data[ids] = torch.randn((len(ids), 2, P, Hkv, D), generator=_gen(3), device=dev, dtype=BF16)
    c = Cache.__new__(Cache)
    c.data, c.arg, c.P, c.layout, c.dev, c.used, c.order = data, data, P, "NHD", dev, 0, ids
    pre, pre_ids = c.runs([330])
    suf, suf_ids = c.runs([100, 64, 200])
    q = torch.randn((3, Hq, D), generator=_gen(4), device=dev, dtype=BF16)
    w = attention.BatchSharedPrefixAttentionWrapper(_ws(dev))
    w.plan(_i32([0, 3], dev), *pre, *suf, *heads, P)
    got = w.run(q, data, return_lse=True)
    d = attention.BatchDecodeWithPagedKVCacheWrapper(_ws(dev), "NHD")
    d.plan(*suf, *heads, P, q_data_type=BF16, window_left=40, first_tokens=3)
    near = d.run(q, data, return_lse=True)
    f = attention.BatchPrefillWithPagedKVCacheWrapper(_ws(dev), "NHD")
    f.plan(_i32([0, 1, 2, 3], dev), *suf, *heads, P, causal=True, q_data_type=BF16, window_left=40, first_tokens=3)
    near2 = f.run(q, data, return_lse=True)
    want, want2 = [], []
    for b, n in enumerate([100, 64, 200]):
        (pk, pv), (sk, sv) = c.tokens(pre_ids[0], 330), c.tokens(suf_ids[b], n)
        want.append(_plain(q[b:b + 1], torch.cat([pk, sk]), torch.cat([pv, sv]), torch.ones((1, 330 + n), dtype=torch.bool, device=dev)))
        t = torch.arange(n, device=dev)[None]
        want2.append(_plain(q[b:b + 1], sk, sv, (t >= n - 41) | (t < 3)))
    _compare(got, _cat(want), "shared")
    _compare(near, _cat(want2), "decode")
    _compare(near2, _cat(want2), "prefill")


# ------------------------------------------------------------------------------- joined states
def _joined(parts, lses):
    lses = lses.double()
    w = torch.nan_to_num(torch.softmax(lses * math.log(2), 0))[..., None]
    p = torch.where(torch.isinf(lses)[..., None], 0.0, parts.double())
    return (w * p).sum(0), (w * p.abs()).sum(0), torch.logsumexp(lses * math.log(2), 0) / math.log(2)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("S,T,H,D", [(1, 1, 1, 64), (2, 5, 32, 128), (3, 1000, 7, 256), (8, 3, 8, 128), (9, 2, 3, 64),
                                     (33, 65, 5, 128), (200, 1, 2, 256), (2, 0, 4, 128), (4, 9000, 16, 64)])
def test_merge_states(dev, dtype, S, T, H, D):
    """Weights and sums in fp32: off by at most (S + 8) 2^-24 relative to sum w|o| (exp2 and the joins), and
    the output's rounding. Parts that saw nothing hold NaN."""
    parts = torch.randn((S, T, H, D), generator=_gen(1), device=dev).to(dtype)
    lses = torch.randn((S, T, H), generator=_gen(2), device=dev) * 20
    none = torch.rand((S, T, H), generator=_gen(3), device=dev) < 0.3
    lses.masked_fill_(none, -math.inf)
    parts.masked_fill_(none[..., None], math.nan)
    out, lse = attention.merge_attention_states(parts, lses)
    want, A, want_lse = _joined(parts, lses)
    assert out.dtype == dtype and out.shape == (T, H, D) and lse.shape == (T, H)
    tol = (S + 8) * 2 ** -22 * A + (2 ** -8 * want.abs() if dtype == BF16 else 0) + 1e-30
    assert not torch.isnan(out).any() and ((out.double() - want).abs() <= tol).all()
    inf = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), inf) and (out[inf] == 0).all()
    assert ((lse.double() - want_lse)[~inf].abs() <= 2 ** -20 + 2 ** -22 * want_lse[~inf].abs()).all()


def test_merge_states_strides_and_aliases(dev):
    S, T, H, D = 3, 11, 4, 128
    wide = torch.randn((T, S, H + 2, D + 8), generator=_gen(1), device=dev, dtype=BF16)
    parts = wide.permute(1, 0, 2, 3)[:, :, 1:-1, :D]
    lses = (torch.randn((H, T, S), generator=_gen(2), device=dev) * 4).permute(2, 1, 0)
    want, A, want_lse = _joined(parts, lses)
    base = attention.merge_attention_states(parts.contiguous(), lses.contiguous())
    got = attention.merge_attention_states(parts, lses)
    assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1])
    _compare(got, (want, A, want_lse), "strided")
    out, lse = attention.merge_attention_states(parts, lses, out=parts[1], lse=lses[2])
    assert out.data_ptr() == parts[1].data_ptr() and torch.equal(out, base[0]) and torch.equal(lses[2], base[1])


def test_infinite_masses(dev):
    """A part of mass 2^inf, and NaN masses, reach the output."""
    parts = torch.ones((2, 3, 1, 64), device=dev)
    lses = torch.tensor([[0.0, math.nan, -math.inf], [1.0, 0.0, math.nan]], device=dev)[..., None]
    out, lse = attention.merge_attention_states(parts, lses)
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1:]).all() and torch.isnan(lse[1:]).all()


# ------------------------------------------------------------------------------- used together
@pytest.mark.parametrize("heads", [(32, 8, 128), (14, 2, 64), (16, 8, 256)])
def test_parts_joined_by_hand_equal_the_whole(dev, heads):
    """A decode step over a shared prefix three ways: the shared wrapper; the prefix by the prefill wrapper
    and the suffixes by the decode wrapper, joined; and one table per request that repeats the prefix."""
    P, sizes, prefix, suffix = 16, [5], 512, [1, 16, 30, 400, 90]
    c, args, kw, q, want = _shared_case(dev, sizes, [prefix], suffix, None, heads, P, seed=8)
    B = len(suffix)
    w = attention.BatchSharedPrefixAttentionWrapper(_ws(dev))
    w.plan(*args, *heads, P)
    shared = w.run(q, c.arg, return_lse=True)
    f = attention.BatchPrefillWithPagedKVCacheWrapper(_ws(dev), "NHD")
    f.plan(_i32([0, B], dev), *args[1:4], *heads, P, causal=False, q_data_type=BF16)
    d = attention.BatchDecodeWithPagedKVCacheWrapper(_ws(dev), "NHD")
    d.plan(*args[4:], *heads, P, q_data_type=BF16)
    parts = torch.empty((2, *q.shape), dtype=BF16, device=dev)
    lses = torch.empty((2, B, heads[0]), device=dev)
    f.run(q, c.arg, out=parts[0], lse=lses[0])
    d.run(q, c.arg, out=parts[1], lse=lses[1])
    joined = attention.merge_attention_states(parts, lses)
    pre, at = args[2].tolist(), args[4].tolist()
    rows = [pre + args[5].tolist()[at[b]:at[b + 1]] for b in range(B)]
    whole = attention.BatchDecodeWithPagedKVCacheWrapper(_ws(dev), "NHD")
    whole.plan(_i32(_cum([len(r) for r in rows]), dev), _i32([i for r in rows for i in r], dev), args[6], *heads, P, q_data_type=BF16)
    _compare(shared, want, "shared")
    _compare(whole.run(q, c.arg, return_lse=True), want, "repeated tables")
    out, A, lse = want
    # (the parts were rounded to bf16 once more before the join: 2^-8 of sum w|o_i| <= A)
    assert ((joined[0].double() - out).abs() <= 2 ** -8 * (2 * A + out.abs()) + 2 ** -11 * A).all()
    assert ((joined[1].double() - lse).abs() <= 2 ** -11 + 2 ** -20 * lse.abs()).all()


def test_a_stream_decoded_in_a_window(dev):
    """Prefill in chunks, then decode steps, of a stream whose window passes over its prompt: each call's
    rows against the definition, on one workspace."""
    heads, P, window, first = (8, 2, 128), 16, 100, 4
    Hq, Hkv, D = heads
    c = Cache(dev, 40, P, Hkv, D, seed=11)
    ids = c.order[:32]
    k, v = c.tokens(ids, 512)
    ws = _ws(dev)
    f, d = attention.BatchPrefillWithPagedKVCacheWrapper(ws, "NHD"), attention.BatchDecodeWithPagedKVCacheWrapper(ws, "NHD")
    at = 0
    for new in (150, 77, 1, 1, 200, 1):
        n = at + new
        pages = -(-n // P)
        tables = (_i32([0, pages], dev), _i32(ids[:pages], dev), _i32([n - P * (pages - 1)], dev))
        q = torch.randn((new, Hq, D), generator=_gen(n), device=dev, dtype=BF16)
        if new > 1:
            f.plan(_i32([0, new], dev), *tables, *heads, P, causal=True, q_data_type=BF16, window_left=window, first_tokens=first)
            got = f.run(q, c.arg, return_lse=True)
        else:
            d.plan(*tables, *heads, P, q_data_type=BF16, window_left=window, first_tokens=first)
            got = d.run(q, c.arg, return_lse=True)
        p, t = torch.arange(at, n, device=dev)[:, None], torch.arange(n, device=dev)[None]
        _compare(got, _plain(q, k[:n], v[:n], (t <= p) & ((t >= p - window) | (t < first))), f"tokens {at}..{n}")
        at = n


def test_native_path_equals_the_general_path(dev, monkeypatch):
    heads = (8, 2, 128)
    c, args, kw, q, _ = _shared_case(dev, [3, 2], [300, 40], [5, 0, 90, 7, 1], None, heads, 16)
    w = attention.BatchSharedPrefixAttentionWrapper(_ws(dev))
    w.plan(*args, *heads, 16)
    d = attention.BatchDecodeWithPagedKVCacheWrapper(_ws(dev), "NHD")
    d.plan(*args[4:], *heads, 16, q_data_type=BF16, window_left=20, first_tokens=2)
    f = attention.BatchPrefillWithPagedKVCacheWrapper(_ws(dev), "NHD")
    f.plan(_i32(range(6), dev), *args[4:], *heads, 16, causal=True, q_data_type=BF16, window_left=20, first_tokens=2)
    out, lse = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty((5, 8), device=dev)
    parts, lses = torch.randn((2, 5, 8, 128), device=dev, dtype=BF16), torch.randn((2, 5, 8), device=dev)
    calls = [lambda x=x, k=k: x.run(q, c.arg, **k) for x in (w, d, f)
             for k in ({}, {"return_lse": True}, {"out": out}, {"out": out, "lse": lse}, {"lse": lse, "return_lse": True})]
    calls += [lambda: attention.merge_attention_states(parts, lses), lambda: attention.merge_attention_states(parts, lses, out, lse)]

    def values(r):
        return [t.clone() for t in (r if isinstance(r, tuple) else (r,))]

    for i, call in enumerate(calls):
        lse.zero_()
        fast = values(call()) + [lse.clone()]
        with monkeypatch.context() as m:
            m.setattr(_lib, "fast", None)
            lse.zero_()
            slow = values(call()) + [lse.clone()]
        assert len(fast) == len(slow) and all(torch.equal(x, y) for x, y in zip(fast, slow)), f"call {i}"


# ------------------------------------------------------------------------------------ refusals
def test_refusals(dev):
    heads = (8, 2, 128)
    c, args, kw, q, _ = _shared_case(dev, [2], [40], [5, 9], None, heads, 16)
    w = attention.BatchSharedPrefixAttentionWrapper(_ws(dev))
    with pytest.raises(RuntimeError, match="plan"):
        w.run(q, c.arg)
    w.plan(*args, *heads, 16)
    for bad in (q[:1], q[:, :4], q.float(), q.transpose(1, 2)):
        with pytest.raises(ValueError):
            w.run(bad, c.arg)
    with pytest.raises(ValueError):
        w.run(q, c.data[:, :, :8])  # another page size
    with pytest.raises(ValueError):
        w.run(q, c.arg, out=torch.empty((3, 8, 128), dtype=BF16, device=dev))
    for lse in (torch.empty((2, 8), dtype=torch.float64, device=dev), torch.empty((8, 2), device=dev),
                torch.empty((2, 16), device=dev)[:, ::2]):
        with pytest.raises(ValueError):
            w.run(q, c.arg, lse=lse)
    with pytest.raises(RuntimeError):
        w.run(q.cpu(), c.arg)
    with pytest.raises(RuntimeError):
        w.run(q, c.arg, lse=torch.empty((2, 8)))
    d = attention.BatchDecodeWithPagedKVCacheWrapper(_ws(dev), "NHD")
    with pytest.raises(ValueError, match="first_tokens"):
        d.plan(*args[4:], *heads, 16, window_left=5, first_tokens=-1)
    with pytest.raises(ValueError, match="first_tokens"):
        d.plan(*args[4:], *heads, 16, window_left=5, first_tokens=2.5)
    parts, lses = torch.zeros((2, 3, 4, 128), dtype=BF16, device=dev), torch.zeros((2, 3, 4), device=dev)
    for p, l in ((parts.half(), lses), (parts[..., :96], lses), (parts[0], lses), (parts, lses[:1]), (parts[:0], lses[:0]),
                 (parts, lses.double()), (parts[..., ::2], lses)):
        with pytest.raises(ValueError):
            attention.merge_attention_states(p, l)
    with pytest.raises(ValueError):
        attention.merge_attention_states(parts, lses, out=torch.empty((3, 4, 128), device=dev))
    with pytest.raises(RuntimeError):
        attention.merge_attention_states(parts, lses.cpu())
    torch.cuda.synchronize()
