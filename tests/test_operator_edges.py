"""Operators without a GPU: calls at the edge of what they accept."""
import pytest
import torch

import tensorjit as tj
from tensorjit.backends.hip_backend import HipProgram
from tensorjit.compiler import lower
from tensorjit.ir import DType, TensorType


def T(*shape, dt="bf16"):
    return TensorType(shape, DType(dt))


def trace(fn, *types):
    return tj.trace(fn, list(types))


CACHE, NEW, PAGES, SEQ = T(10, 4, 3, 24), T(2, 5, 3, 24), T(2, 6, dt="i32"), T(2, dt="i32")


# ---------------------------------------------------------------------------
# writes in place
# ---------------------------------------------------------------------------


def test_a_write_does_not_read_its_own_cache():
    """As it is, reshaped on either side, through two reshapes, and of a write's result."""
    def same(c, x, p, s):
        return tj.paged_write(c, c, p, s)

    def rows(c, x, p, s):
        return tj.paged_write(c, tj.reshape(c, 2, 20, 3, 24), p, s)

    def cache(c, x, p, s):
        return tj.paged_write(tj.reshape(c, 10, 4, 3, 24), c, p, s)

    def both(c, x, p, s):
        return tj.paged_write(tj.reshape(c, 10, 4, 3, 24), tj.reshape(tj.reshape(c, 40, 72), 2, 20, 3, 24), p, s)

    def chained(c, x, p, s):
        first = tj.paged_write(c, x, p, s)
        return tj.paged_write(first, tj.reshape(first, 2, 20, 3, 24), p, s)

    def chained_cache(c, x, p, s):
        first = tj.paged_write(c, x, p, s)
        return tj.paged_write(tj.reshape(first, 10, 4, 3, 24), tj.reshape(first, 2, 20, 3, 24), p, s)

    as_rows = T(2, 20, 3, 24)
    for fn, kind in ((same, as_rows), (rows, CACHE), (cache, as_rows), (both, CACHE), (both, T(10, 4, 72)), (chained, CACHE),
                     (chained_cache, CACHE)):
        with pytest.raises(ValueError, match="read the result"):
            lower(trace(fn, kind, NEW, PAGES, SEQ))


def test_a_reshaped_cache_is_written_once():
    """Reshapes of the destination alone stay allowed."""
    def f(c, x, p, s):
        first = tj.paged_write(tj.reshape(c, 10, 4, 3, 24), x, p, s)
        return tj.paged_write(tj.reshape(tj.reshape(first, 40, 72), 10, 4, 3, 24), x + 1.0, p, s)

    program = lower(trace(f, T(10, 4, 72), NEW, PAGES, SEQ))
    assert program.storage(program.graph.outputs[0]) is program.graph.inputs[0]


# ---------------------------------------------------------------------------
# number parameters: fp32 constants of the kernels
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("scale", [5e-324, 1e-46, 1e-38, 9e-31, 1.1e30])
def test_paged_attention_refuses_scales_that_fp32_does_not_hold(scale):
    """A scale that is 0 in fp32 makes a masked score, -inf, times it NaN."""
    with pytest.raises(ValueError, match="paged_attention: scale"):
        trace(lambda q, c, p, s: tj.paged_attention(q, c, c, p, s, scale=scale), T(2, 5, 6, 24), CACHE, PAGES, SEQ)


@pytest.mark.parametrize("magnitude", [1e-46, -1e-46, 1e-40, -9e-31])
def test_rotary_refuses_magnitudes_that_fp32_does_not_hold(magnitude):
    """1e-46 is 0 in fp32, and 1e-40 keeps half of its digits; 0 itself is one."""
    def rotary(m):
        return trace(lambda x, p: tj.rotary(x, p, magnitude=m), NEW, T(2, 5, dt="i32"))

    with pytest.raises(ValueError, match="rotary: magnitude"):
        rotary(magnitude)
    assert rotary(0).outputs[0].type == NEW and rotary(-1e-30).outputs[0].type == NEW


@pytest.mark.parametrize("temperature", [5e-324, 1e-300, 7e-46])
def test_sample_refuses_temperatures_that_are_zero_in_fp32(temperature):
    """As 0 they would give the first of several largest logits instead of one of them by its share."""
    def sample(t):
        return trace(lambda x, u: tj.sample(x, u, temperature=t), T(3, 50), T(3, dt="f32"))

    with pytest.raises(ValueError, match="sample: temperature"):
        sample(temperature)
    for t in (0, 0.0, -0.0, 1e-38, 1.5e-45):
        assert sample(t).outputs[0].type == TensorType((3,), DType.i32)


def test_refusals_do_not_depend_on_how_denormals_are_handled():
    """A library built with -ffast-math has its process flush them (this repository's oracle is one)."""
    tiny = 5e-324
    flushed = tiny * 1.0 == 0.0
    torch.set_flush_denormal(True)
    try:
        with pytest.raises(ValueError, match="sample: temperature"):
            trace(lambda x, u: tj.sample(x, u, temperature=tiny), T(3, 50), T(3, dt="f32"))
        with pytest.raises(ValueError, match="rotary: magnitude"):
            trace(lambda x, p: tj.rotary(x, p, magnitude=-tiny), NEW, T(2, 5, dt="i32"))
    finally:
        torch.set_flush_denormal(flushed)


# ---------------------------------------------------------------------------
# calls
# ---------------------------------------------------------------------------


def program_of(fn, *types):
    """A program's argument checks, on CPU tensors and without its kernels."""
    program = object.__new__(HipProgram)
    program.program = lower(trace(fn, *types))
    program._input_index = {id(n): i for i, n in enumerate(program.program.graph.inputs)}
    program._out_nodes, program._out_index, program.device_index = [], {}, 0
    program._init_call_path()
    program.device_index = -1           # where tensors of the CPU are
    return program


def test_torch_sees_writes_in_place():
    """What autograd saved of a cache before it was written is refused in the backward pass."""
    program = program_of(lambda c, x, p, s: tj.paged_write(c, x, p, s), T(10, 4, 3, 24, dt="f32"), T(2, 5, 3, 24, dt="f32"), PAGES, SEQ)
    cache, new = torch.zeros(10, 4, 3, 24), torch.zeros(2, 5, 3, 24)
    args = [cache, new, torch.zeros(2, 6, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)]
    w = torch.ones(24, requires_grad=True)
    loss = (w * cache).sum()
    before = [t._version for t in args]
    program._prepare(args)
    assert cache._version > before[0] and [t._version for t in args[1:]] == before[1:]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        args[0] = torch.zeros(10, 4, 3, 24)         # has no counter
    program._prepare(args)
