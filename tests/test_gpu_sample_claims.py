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


@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("n", [5003, 65521, 248320])
def test_sample_of_a_row_in_any_batch(ops, n, dtype):
    """The same row, alone and among others of batches that take other clusters and forms, wherever it starts: the same token."""
    gen = torch.Generator(device=DEV).manual_seed(n)
    few = 12
    x = (torch.randn(few, n, generator=gen, device=DEV) * 2).to(dtype)
    u = torch.rand(few, generator=gen, device=DEV)
    t = torch.empty(few, device=DEV).uniform_(0.5, 1.5, generator=gen)
    k = torch.tensor([0, 50, 0, 0, 400, 3, 0, 200, 0, 0, 5000, 1], dtype=torch.int32, device=DEV)
    p = torch.tensor([0.9, 1.0, 0.5, 1.0, 0.95, 0.9, 0.99, 0.3, 1.0, 0.8, 0.9, 1.0], device=DEV)
    m = torch.tensor([0.0, 0.0, 0.0, 0.01, 0.0, 0.2, 1e-4, 0.0, 0.0, 1e-6, 0.0, 0.0], device=DEV)
    alone = torch.cat([ops.sample_rows(x[i: i + 1], u[i: i + 1], *(v[i: i + 1] for v in (t, k, p, m))) for i in range(few)])
    assert torch.equal(alone.cpu(), sample64(x, u, t, k, p, m))
    for rows in (12, 24, 40, 72, 150, 300):
        pick = torch.randint(few, (rows,), generator=gen, device=DEV)
        wide = torch.empty(rows, n + 5, dtype=dtype, device=DEV)
        wide[:, 3: n + 3] = x[pick]
        got = ops.sample_rows(wide[:, 3: n + 3], u[pick], t[pick], k[pick], p[pick], m[pick])
        assert torch.equal(got, alone[pick])


def test_sample_under_no_temperature(ops):
    """NaN, zero and less take the largest, whatever else is asked for; so does the row beside them that asks for it by top_k."""
    x = torch.randn(5, 70001, generator=torch.Generator().manual_seed(3)).to(DEV)
    x[:, [17, 60000]] = 9.0
    u = torch.full((5,), 0.99, device=DEV)
    t = torch.tensor([NAN, 0.0, -3.0, -INF, 1.0], device=DEV)
    k = torch.tensor([0, 50, 3000, 0, 1], dtype=torch.int32, device=DEV)
    assert ops.sample_rows(x, u, t, k, 0.9, 0.01).tolist() == [17] * 5
    assert ops.sample_rows(x, u, NAN).tolist() == [17] * 5
