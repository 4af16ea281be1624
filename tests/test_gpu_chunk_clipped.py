"""Sequences of which the packed rows hold a part only: append and attention agree on where a token stands."""
import pytest
import torch

from chunk_helpers import BF, attention64, attention_tolerance, cached_rows, make_batch, sequences

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from b200attn import ops
    return ops


# (new, held, rows that are not there, kv heads, group, head size): few rows a sequence, and many
CLIPPED = [([5, 3], [20, 0], 2, 2, 4, 256), ([9, 1, 2], [300, 41, 7], 7, 2, 2, 128), ([90, 40], [333, 64], 7, 2, 4, 256),
           ([300, 20], [1500, 2], 260, 4, 3, 128), ([130], [15], 129, 1, 7, 256)]


@pytest.mark.parametrize("new,held,gone,hkv,group,dim", CLIPPED)
def test_first_sequence_begins_in_front_of_the_rows(ops, new, held, gone, hkv, group, dim):
    """cu_seqlens[0] = -gone: row t is token t + gone of its sequence, whose first `gone` are in the cache already."""
    t = make_batch(new, held, hkv, group, dim, seed=gone, device=DEV, junk=0.0)
    want, spread = attention64(t, t["gate"])
    u = t | dict(q=t["q"][gone:], gate=t["gate"][gone:], cu=t["cu"] - gone)
    out = ops.paged_gqa_attention_chunk(u["q"], u["k_cache"], u["v_cache"], u["table"], u["cu"], u["pos"], gate=u["gate"])
    assert out.shape[0] == sum(new) - gone > 0
    worst = ((out.double() - want[gone:]).abs() / attention_tolerance(want, spread)[gone:]).max().item()
    assert worst <= 1, worst
    # appended to where the attention looks for them: the caches come out as they were
    freq = torch.zeros(32, device=DEV)                      # angle 0: keys go in as they are
    k, v = torch.empty_like(t["k"]), torch.empty_like(t["v"])
    for b, (n, h) in enumerate(zip(new, held)):
        first = sum(new[:b])
        k[first: first + n] = cached_rows(t["k_cache"], t["table"], b, n + h)[h:].to(BF)
        v[first: first + n] = cached_rows(t["v_cache"], t["table"], b, n + h)[h:].to(BF)
    kc, vc = t["k_cache"].clone(), t["v_cache"].clone()
    ops.paged_kv_append_rope(u["q"], k[gone:], v[gone:], kc, vc, u["table"], u["cu"], u["pos"],
                             torch.arange(out.shape[0], device=DEV), freq, 64)
    assert torch.equal(kc, t["k_cache"]) and torch.equal(vc, t["v_cache"])


@pytest.mark.parametrize("cu", [[150, 100, 200], [40, 0, 200, 90], [199, 120, 60, 1, 200]])
def test_lengths_that_do_not_ascend_touch_no_held_token(ops, cu):
    """Not a call with a meaning, but what sequences hold already stays as it is."""
    held = [300] * (len(cu) - 1)
    t = make_batch([200] * len(held), held, 2, 4, 256, seed=len(cu), device=DEV, junk=0.0, cached=False)
    before = t["k_cache"].clone(), t["v_cache"].clone()
    ops.paged_kv_append_rope(t["q"][:200], t["k"][:200], t["v"][:200], t["k_cache"], t["v_cache"], t["table"],
                             torch.tensor(cu, dtype=torch.int32, device=DEV), t["pos"], torch.arange(200, device=DEV), torch.ones(32, device=DEV), 64)
    for b, h in enumerate(held):
        for cache, old in zip((t["k_cache"], t["v_cache"]), before):
            assert torch.equal(cached_rows(cache, t["table"], b, h), cached_rows(old, t["table"], b, h))


@pytest.mark.parametrize("new,held,rows,hkv,group,dim", [([5, 3], [20, 0], 6, 2, 4, 256), ([2, 3, 9], [300, 41, 7], 4, 2, 2, 128),
                                                         ([90, 40], [333, 64], 70, 2, 4, 256), ([100, 500, 400], [20, 1500, 3], 190, 4, 3, 128)])
def test_lengths_that_name_more_rows_than_there_are(ops, new, held, rows, hkv, group, dim):
    """The rows that are there come out as in the whole batch, and they alone are appended."""
    t = make_batch(new, held, hkv, group, dim, seed=rows, device=DEV, junk=0.0)
    want, spread = attention64(t, t["gate"])
    out = ops.paged_gqa_attention_chunk(t["q"][:rows], t["k_cache"], t["v_cache"], t["table"], t["cu"], t["pos"], gate=t["gate"][:rows])
    worst = ((out.double() - want[:rows]).abs() / attention_tolerance(want, spread)[:rows]).max().item()
    assert out.shape[0] == rows and worst <= 1, worst
    vc = t["v_cache"].clone()
    ops.paged_kv_append_rope(t["q"][:rows], t["k"][:rows], t["v"][:rows], t["k_cache"].clone(), vc, t["table"], t["cu"], t["pos"],
                             torch.arange(rows, device=DEV), torch.ones(32, device=DEV), 64)
    for b, first, n, h in sequences(t):
        there = max(0, min(n, rows - first))
        got, old = cached_rows(vc, t["table"], b, h + n), cached_rows(t["v_cache"], t["table"], b, h + n)
        assert torch.equal(got[h: h + there], t["v"][first: first + there].double())
        assert torch.equal(got[:h], old[:h]) and torch.equal(got[h + there:], old[h + there:])
