"""The operators on the GPU, for calls at the edge of what they accept, against their definitions in float64."""
import math

import pytest
import torch

import operator_reference as ref
import tensorjit as tj

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _env(monkeypatch, tmp_path_factory):
    if not (torch.cuda.is_available() and torch.version.hip):
        pytest.skip("needs a ROCm GPU")
    monkeypatch.setenv("TENSORJIT_NO_AUTOTUNE", "1")
    monkeypatch.setenv("TENSORJIT_CACHE_DIR", str(tmp_path_factory.getbasetemp() / "tjcache"))


def gen(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(*shape, dt=torch.float32, seed=0, scale=1.0):
    return (scale * torch.randn(shape, device=DEV, generator=gen(seed))).to(dt)


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------


def mass_error(logits, temperature):
    """How far a cumulative mass may be off, of the total, which is at least the largest mass: per token
    half a step of 2^-43 of that; and of each mass the exponential's 2^-38 and what 64-bit arithmetic
    makes of the exponent, 2^-52 of the largest logit over the temperature, in either's unit."""
    x = logits.double()
    x = x[x.isfinite()]
    t = float(torch.as_tensor(temperature, dtype=torch.float64).min())
    size = float(x.abs().max()) / t if x.numel() and t > 0 else 0.0
    return logits.shape[-1] * 2.0**-44 + 2.0**-38 + size * 2.0**-52


def check_sample(logits, uniform, aside=0, **params):
    """``aside``: rows that may stand nearer to a border than two sums (of either side) may be off."""
    tensors = {n: p for n, p in params.items() if isinstance(p, torch.Tensor)}

    def fn(x, u, *rest):
        return tj.sample(x, u, **{**params, **dict(zip(tensors, rest))})

    got = tj.jit(fn)(logits, uniform, *tensors.values())
    want, margin = ref.sample(logits, uniform, **params)
    clear = margin > 2 * mass_error(logits, params.get("temperature", 1.0))
    assert int((~clear).sum()) <= aside
    assert torch.equal(got.cpu()[clear], want[clear])
    return got


@pytest.mark.parametrize("V", [300, 70000])
@pytest.mark.parametrize("size", [1e-33, 1e-36])
def test_sample_small_temperatures(V, size):
    """Logits as small as the temperature: their quotient counts, whatever its parts."""
    R = 6
    x, u = normal(R, V, scale=3.0) * size, torch.rand(R, device=DEV, generator=gen(1))
    t = (0.5 + torch.rand(R, device=DEV, generator=gen(5))) * size
    check_sample(x, u, aside=1, temperature=t)
    check_sample(x, u, aside=1, temperature=t, top_p=0.8)
    check_sample(x, u, aside=1, temperature=t, top_k=40, min_p=0.01)
    check_sample(x, u, aside=1, temperature=size)


# ---------------------------------------------------------------------------
# writes in place
# ---------------------------------------------------------------------------


def test_torch_sees_writes_in_place():
    """A call, an eager one and one under capture, moves the version of the cache and of nothing else."""
    cache, x = normal(6, 4, 2, 8), normal(2, 3, 2, 8, seed=1)
    pages = torch.arange(6, dtype=torch.int32, device=DEV).reshape(2, 3)
    starts = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    args = (cache, x, pages, starts)
    f = tj.jit(lambda *a: tj.paged_write(*a))
    f(*args)
    w = torch.ones(8, device=DEV, requires_grad=True)
    loss = (w * cache).sum()
    before = [t._version for t in args]
    assert f(*args) is cache
    assert cache._version > before[0] and [t._version for t in args[1:]] == before[1:]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    before, graph = cache._version, torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f(*args)
    assert cache._version > before
    with torch.inference_mode():
        other = cache.clone().zero_()
        assert f(other, x, pages, starts) is other
    want = ref.paged_write(torch.zeros(6, 4, 2, 8), x.cpu(), pages.cpu(), starts.cpu())
    assert torch.equal(other.cpu(), want)
