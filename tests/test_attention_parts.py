"""CPU: plans of the attention wrappers over parts of a cache refuse bad tables before any launch, and
runs refuse tensors off the GPU."""
from __future__ import annotations

import pytest
import torch

from pie_amd import attention

HEADS = (8, 2, 128)


def _i32(*xs):
    return torch.tensor(xs, dtype=torch.int32)


def _tables(**kw):
    """Two groups of one and two requests."""
    t = dict(group_indptr=_i32(0, 1, 3), prefix_indptr=_i32(0, 2, 3), prefix_indices=_i32(4, 5, 6),
             prefix_last_page_len=_i32(3, 16), paged_kv_indptr=_i32(0, 1, 1, 3), paged_kv_indices=_i32(0, 1, 2),
             paged_kv_last_page_len=_i32(1, 0, 7))
    t.update(kw)
    return t


def _plan(ws=1 << 24, heads=HEADS, page=16, **kw):
    w = attention.BatchSharedPrefixAttentionWrapper(torch.zeros(ws, dtype=torch.uint8))
    w.plan(**_tables(**{k: v for k, v in kw.items() if k != "qo_indptr"}), num_qo_heads=heads[0], num_kv_heads=heads[1],
           head_dim=heads[2], page_size=page, qo_indptr=kw.get("qo_indptr"))
    return w


def test_a_plan_knows_its_work():
    w = _plan()
    p = w._plan
    assert p["T"] == 3 and p["info"][2] + p["info"][4] == 2 and p["plan"].numel() == p["info"][0]
    assert _plan(qo_indptr=_i32(0, 1, 1, 4))._plan["T"] == 4
    with pytest.raises(RuntimeError, match="GPU"):
        w.run(torch.zeros((3, 8, 128), dtype=torch.bfloat16), torch.zeros((8, 2, 16, 2, 128), dtype=torch.bfloat16))


@pytest.mark.parametrize("bad", [
    dict(group_indptr=_i32(0, 1, 2)),               # a request outside every group
    dict(group_indptr=_i32(1, 1, 3)),
    dict(group_indptr=_i32(0, 4, 3)),
    dict(group_indptr=_i32(0, 3)),                  # another number of groups
    dict(prefix_indptr=_i32(0, 2, 1)),
    dict(prefix_indptr=_i32(0, 2, 9)),              # more pages than ids
    dict(prefix_last_page_len=_i32(17, 16)),
    dict(prefix_last_page_len=_i32(-1, 16)),
    dict(paged_kv_indptr=_i32(0, 2, 1, 3)),
    dict(paged_kv_indptr=_i32(0, 1, 1, 9)),
    dict(paged_kv_last_page_len=_i32(1, 0, 99)),
    dict(paged_kv_indptr=torch.tensor([0, 1, 1, 3])),  # int64
    dict(qo_indptr=_i32(1, 1, 1, 4)),
    dict(qo_indptr=_i32(0, 2, 1, 4)),
    dict(qo_indptr=_i32(0, 2, 4)),
    dict(heads=(8, 3, 128)), dict(heads=(8, 0, 128)), dict(heads=(64, 2, 128)), dict(heads=(8, 2, 96)),
    dict(page=0), dict(ws=1000),
])
def test_bad_tables_are_refused(bad):
    with pytest.raises(ValueError):
        _plan(**bad)


def test_first_tokens_are_whole_numbers():
    ws = torch.zeros(1 << 20, dtype=torch.uint8)
    d, f = attention.BatchDecodeWithPagedKVCacheWrapper(ws), attention.BatchPrefillWithPagedKVCacheWrapper(ws)
    t = (_i32(0, 1), _i32(0), _i32(9))
    for bad in (-1, 1.5, True):
        with pytest.raises(ValueError, match="first_tokens"):
            d.plan(*t, *HEADS, 16, window_left=3, first_tokens=bad)
        with pytest.raises(ValueError, match="first_tokens"):
            f.plan(_i32(0, 2), *t, *HEADS, 16, window_left=3, first_tokens=bad)


def test_merge_refuses_tensors_off_the_gpu():
    with pytest.raises(RuntimeError, match="GPU"):
        attention.merge_attention_states(torch.zeros((2, 1, 1, 64)), torch.zeros((2, 1, 1)))
