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
    """How far one mass may be off, of the largest (half a step of 2^-43) and of itself: the exponential's 2^-38, and what
    64-bit arithmetic makes of the exponent, 2^-52 of the largest logit over the temperature, in either's unit."""
    x = logits.double()
    x = x[x.isfinite()]
    t = float(torch.as_tensor(temperature, dtype=torch.float64).min())
    size = float(x.abs().max()) / t if x.numel() and t > 0 else 0.0
    return 2.0**-44, 2.0**-38 + size * 2.0**-52


def clear_of_borders(logits, uniform, errors, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """Whether each row's choice is the same wherever its masses lie within their errors.  A sum of V masses is off
    by V times the first error and once the second, of the row's total, which is at least the largest mass; two
    sums are compared.  ``min_p`` is compared with one mass."""
    step, relative = errors
    two_sums = 2 * (logits.shape[-1] * step + relative)

    def at(p, r):
        return None if p is None else float(p[r]) if isinstance(p, torch.Tensor) else float(p)

    clear = []
    for r, x in enumerate(logits.detach().cpu().double()):
        t, k, tp, mp = (at(v, r) for v in (temperature, top_k, top_p, min_p))
        if not t > 0:
            clear.append(True)
            continue
        p = torch.exp((x - x.max()) / t)
        order = torch.argsort(x, descending=True, stable=True)
        keep, ok = order[:int(k)] if k is not None and k > 0 else order, True
        if tp is not None and tp < 1:
            upto = p[keep].cumsum(0)
            ok &= bool(((upto[:-1] - tp * upto[-1]).abs() > two_sums * upto[-1]).all())
            keep = keep[:1 + int((upto < tp * upto[-1]).sum())]
        if mp is not None:
            others = p[keep][p[keep] < 1]
            ok &= bool(((others - mp).abs() > step + relative * others).all())
            keep = keep[p[keep] >= mp]
        upto = p[keep.sort().values].cumsum(0)
        ok &= bool(((upto[:-1] - float(uniform[r]) * upto[-1]).abs() > two_sums * upto[-1]).all())
        clear.append(ok)
    return torch.tensor(clear)


def check_sample(logits, uniform, aside=0, **params):
    """``aside``: rows that may stand on a border."""
    tensors = {n: p for n, p in params.items() if isinstance(p, torch.Tensor)}

    def fn(x, u, *rest):
        return tj.sample(x, u, **{**params, **dict(zip(tensors, rest))})

    got = tj.jit(fn)(logits, uniform, *tensors.values())
    want = ref.sample(logits, uniform, **params)[0]
    clear = clear_of_borders(logits, uniform, mass_error(logits, params.get("temperature", 1.0)), **params)
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


def two_values(dt, R, V, top_k=None, top_p_at=None, min_p=None):
    """Rows with every seventh logit 1 and the others 0, uniforms in the middle of a kept token's
    share, and ``top_p`` in the middle of the share of the token ``top_p_at`` (in order): no row
    stands on a border.  The filters in float64, from counts alone."""
    x = torch.zeros(R, V)
    x[:, ::7] = 1.0
    p = torch.exp(x[0].double() - 1.0)
    order = torch.cat([torch.arange(0, V, 7), torch.tensor([i for i in range(V) if i % 7])])
    kept, top_p = order[:top_k], None
    if top_p_at is not None:
        cum = p[kept].cumsum(0)
        top_p = float(((cum[top_p_at] - p[kept[top_p_at]] / 2) / cum[-1]).float())
        kept = kept[:top_p_at + 1]
    if min_p is not None:
        kept = kept[p[kept] >= min_p]
    kept = kept.sort().values
    cum = p[kept].cumsum(0)
    at = torch.tensor([0, len(kept) - 1, len(kept) // 2, len(kept) // 3])[:R]
    u = ((cum[at] - p[kept[at]] / 2) / cum[-1]).float()
    # as one value per row, those that mean all tokens among them: one program serves every case
    params = dict(top_k=torch.full((R,), top_k or 0, dtype=torch.int32, device=DEV),
                  top_p=torch.full((R,), top_p or 1.0, device=DEV), min_p=torch.full((R,), min_p or 0.0, device=DEV))
    return x.to(DEV, dt), u.to(DEV), params, kept[at]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [9001, 100003, 151001])
def test_sample_borders_within_equal_logits(dt, V):
    """A filter ends among thousands of equal logits, more than are ranked: by their keys' digits and
    then by index, for rows of one workgroup and rows split over several.  Every row is compared."""
    ones = -(-V // 7)
    for kwargs in (dict(top_k=300), dict(top_k=ones), dict(top_k=V // 3), dict(top_k=V - 1), dict(top_p_at=200), dict(top_p_at=ones - 1),
                   dict(top_p_at=ones + 4321), dict(top_k=V // 2, top_p_at=V // 3), dict(top_k=V // 2, top_p_at=77),
                   dict(top_k=V // 3, min_p=0.5), dict(top_p_at=V // 2, min_p=0.3), dict(min_p=0.5)):
        x, u, params, want = two_values(dt, 4, V, **kwargs)
        got = check_sample(x, u, **params)
        assert got.tolist() == want.tolist(), kwargs


@pytest.mark.parametrize("V", [100003, 1 << 20])
def test_sample_long_rows_by_the_bound_of_their_length(V):
    """Cumulative masses are off by up to V half steps, so which rows are set aside follows from V.  At 2^20
    tokens a nucleus of 0.999 ends among masses smaller than that; one row of three is always compared."""
    R = 3
    x, u = normal(R, V, scale=3.0), torch.rand(R, device=DEV, generator=gen(1))
    k = torch.tensor([0, 700, V // 4], dtype=torch.int32, device=DEV)
    p = torch.tensor([0.95, 0.5, 0.999], device=DEV)
    for params in (dict(), dict(top_k=k), dict(top_p=p), dict(top_k=k, top_p=p), dict(min_p=1e-4)):
        check_sample(x, u, aside=2, **params)


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


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


def caches(B, L, page, KV, D, dt, seed=0, scale=1.0):
    """K, V and a page table whose sequences own distinct, shuffled pages."""
    P = -(-L // page)
    pages = torch.randperm(B * P, device=DEV, generator=gen(seed)).reshape(B, P).to(torch.int32)
    return normal(B * P, page, KV, D, dt=dt, seed=seed, scale=scale), normal(B * P, page, KV, D, dt=dt, seed=seed + 1), pages


@pytest.mark.parametrize("dt, size", [(torch.float16, 3e3), (torch.float16, 1e4), (torch.bfloat16, 3e3), (torch.bfloat16, 1e5),
                                      (torch.bfloat16, 1e15), (torch.float32, 1e5), (torch.float32, 1e15)])
@pytest.mark.parametrize("S", [1, 6, 70])
@pytest.mark.parametrize("negative", [False, True])
def test_scores_of_any_size(dt, size, S, negative):
    """Scores that fp32 holds give what they give in 64 bits: the value of the largest one's key, where the next is
    20 and more below it, whatever 64 products in fp32 may be off."""
    B, L, D = 2, 300, 64
    k, v, pages = caches(B, L, 16, 2, D, dt, scale=size)
    if negative:                     # every score far below zero
        k[..., 0] = 4.0 * size
    q = normal(B, S, 6, D, dt=dt, seed=5, scale=size)
    if negative:
        q[..., 0] = -6.0 * size
    assert q.isfinite().all() and k.isfinite().all()
    starts = torch.tensor([L - S, 40], dtype=torch.int32, device=DEV)
    got = tj.jit(lambda *a: tj.paged_attention(*a))(q, k, v, pages, starts)
    compared = 0
    for b in range(B):
        ks, vs = (t[pages[b].long()].flatten(0, 1).double() for t in (k, v))
        for i in range(S):
            n = int(starts[b]) + i + 1
            for h in range(6):
                x = q[b, i, h].double()
                s, terms = ks[:n, h // 3] @ x / 8, ks[:n, h // 3].abs() @ x.abs() / 8
                top = s.topk(2)
                if float(top.values[0] - top.values[1]) < 20 + 2 * 66 * 2.0**-24 * float(terms.max()):
                    continue
                compared += 1
                want = vs[top.indices[0], h // 3]
                assert bool(((got[b, i, h].double() - want).abs() <= torch.finfo(dt).eps * want.abs() + 2.0**-24).all()), (b, i, h)
    assert compared > B * S * 3
    assert got.isfinite().all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("S, G, L", [(1, 4, 40000), (24, 4, 5000), (3, 2, 5000)])
@pytest.mark.parametrize("lead", [5.0, 12.0, 18.0])
def test_many_keys_behind_one_that_leads(dt, S, G, L, lead):
    """One key's score is above all others by ``lead`` and its value is zero, so the output is what the small
    weights of the others add up to.  fp16 holds a weight (at most half a step of its own size, as in every
    bound) or half of 2^-31 of the largest, which the reference of a row is never above."""
    D, page, KV = 64, 16, 2
    P = -(-L // page)
    k, v = torch.zeros(P, page, KV, D, device=DEV), 1.0 + torch.rand(P, page, KV, D, device=DEV, generator=gen(1))
    k[..., 1] = torch.randn(P, page, KV, device=DEV, generator=gen(2)) * 0.25      # other scores: -0.25 .. 0.25 or so
    k[L // 3 // page, L // 3 % page, :, 0] = 8.0
    v[L // 3 // page, L // 3 % page] = 0.0
    q = torch.zeros(2, S, KV * G, D, device=DEV)
    q[..., 0], q[..., 1] = lead, 1.0
    q, k, v = (t.to(dt) for t in (q, k, v))
    pages = torch.arange(P, dtype=torch.int32, device=DEV).expand(2, P).contiguous()
    starts = torch.tensor([L - S, L // 2], dtype=torch.int32, device=DEV)
    got = tj.jit(lambda *a: tj.paged_attention(*a))(q, k, v, pages, starts).cpu().double()
    want, bound = ref.paged_attention(q, k, v, pages, starts)
    if dt == torch.float16:
        n = starts.cpu().double()[:, None, None, None] + S
        bound = bound + n * 2.0**-32 * float(v.abs().max()) + 2.0**-25      # and the output's own smallest step
    assert bool((want > 0).all()) and bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / want).max())
