"""How far a key or value that is no number reaches among the new tokens of a call."""
import pytest
import torch

from chunk_helpers import make_batch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BLOCK = 256                                     # most tokens that share a block


@pytest.fixture(scope="module")
def ops():
    from b200attn import ops
    return ops


def attend(ops, t):
    return ops.paged_gqa_attention_chunk(t["q"], t["k_cache"], t["v_cache"], t["table"], t["cu"], t["pos"], gate=t["gate"])


def place(t, b, index):
    return int(t["table"][b, index // 16]), index % 16


# sequence 0's token `at` is spoiled: few rows a sequence, and many
SPOILED = [([4, 3], [40, 17], 2), ([1, 2, 1], [16, 600, 31], 0), ([700, 60], [300, 90], 650), ([300, 300], [1000, 5], 299), ([2000, 3], [30, 8], 1500)]


@pytest.mark.parametrize("new,held,at", SPOILED)
@pytest.mark.parametrize("hkv,group,dim", [(2, 4, 256), (3, 1, 128)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_a_spoiled_key_reaches_the_tokens_that_see_it(ops, new, held, at, hkv, group, dim, value):
    t = make_batch(new, held, hkv, group, dim, seed=at, device=DEV)
    want = attend(ops, t)
    page, slot = place(t, 0, held[0] + at)
    t["k_cache"][page, :, slot] = value
    got = attend(ops, t)
    assert torch.equal(got[:at], want[:at]) and torch.equal(got[new[0]:], want[new[0]:])
    assert torch.isfinite(got[:at].float()).all()


@pytest.mark.parametrize("new,held,at", SPOILED)
@pytest.mark.parametrize("hkv,group,dim", [(2, 4, 256), (3, 1, 128)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_spoiled_value_reaches_its_block_and_no_further(ops, new, held, at, hkv, group, dim, value):
    t = make_batch(new, held, hkv, group, dim, seed=at, device=DEV)
    want = attend(ops, t)
    page, slot = place(t, 0, held[0] + at)
    t["v_cache"][page, :, slot] = value
    got = attend(ops, t)
    safe = max(0, at - (BLOCK - 1))
    assert torch.equal(got[:safe], want[:safe]) and torch.equal(got[new[0]:], want[new[0]:])
    assert not torch.isfinite(got[at].float()).any()
