"""What the documentation of `sample_rows` says of parameters at the ends of their range, and of a row in any batch."""
import pytest
import torch

from chunk_helpers import BF, sample64

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = float("inf"), float("nan")
KEEP_ALL = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}


@pytest.fixture(scope="module")
def ops():
    from b200attn import ops
    return ops


@pytest.mark.parametrize("kwargs", [dict(), dict(top_k=4), dict(top_k=900), dict(top_p=0.6), dict(min_p=0.4), dict(top_k=40, top_p=0.9, min_p=1e-3)])
@pytest.mark.parametrize("temperature", [1e36, 4e36, 1e38, 3.4e38])
def test_sample_under_the_largest_temperatures(ops, temperature, kwargs):
    """Logits over the whole range of the type, of which such a temperature makes weights that still differ."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(6, 5003, generator=gen)
    x[0] *= 1e37
    x[1] = x[1].clamp(-3, 3) * 1e38
    x[2] = -1e30 + x[2]
    x[3] = torch.rand(5003, generator=gen) * 3.4e38
    x[4, ::2] = torch.finfo(torch.float32).min
    x, u = x.to(DEV), torch.rand(6, generator=gen).to(DEV)
    want = sample64(x, u, **(KEEP_ALL | kwargs | {"temperature": temperature}))
    assert torch.equal(ops.sample_rows(x, u, temperature, **kwargs).cpu(), want)


@pytest.mark.parametrize("kwargs", [dict(), dict(top_k=7, top_p=0.9)])
def test_sample_under_an_infinite_temperature(ops, kwargs):
    """Counts as the largest float, under which ordinary logits all weigh the same."""
    x = torch.randn(4, 999, generator=torch.Generator().manual_seed(2)).to(DEV)
    u = torch.tensor([0.0, 0.3, 0.5, 0.999], device=DEV)
    want = sample64(x, u, **(KEEP_ALL | kwargs | {"temperature": INF}))
    assert torch.equal(ops.sample_rows(x, u, INF, **kwargs).cpu(), want)
    assert torch.equal(ops.sample_rows(x, u, torch.full((4,), INF, device=DEV), **kwargs).cpu(), want)
