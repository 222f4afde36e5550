"""rotary against its definition in fp64, over types, layouts, axes and far positions."""

import pytest
import torch

from cs348k_fast_attention_grammar_b200 import FaError, rotary
from paged_reference import assert_within, rotary_tolerance, rotate

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _x(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


def _freq(R, base=10000.0, dtype=torch.float32):
    return (base ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,H,S,D,R", [(1, 1, 1, 16, 16), (2, 3, 5, 64, 64), (1, 5, 257, 80, 32),
                                       (3, 2, 33, 128, 128), (1, 48, 3, 256, 96),
                                       (1, 2, 40, 24, 16), (1, 40, 7, 1024, 1024)])
def test_matches_definition(dtype, interleaved, B, H, S, D, R):
    x, f = _x((B, H, S, D), dtype), _freq(R)
    pos = torch.randint(0, 5000, (B, S), generator=torch.Generator().manual_seed(1)).to(DEV)
    for inverse in (False, True):
        got = rotary(x, pos, f, interleaved=interleaved, inverse=inverse)
        want, size = rotate(x, (pos.double()[..., None] * f.double())[:, None], interleaved, inverse)
        assert_within(got, want, rotary_tolerance(want, size, dtype), f"{D}/{R} {inverse}")
        assert torch.equal(got[..., R:], x[..., R:])


@pytest.mark.parametrize("sections", [(8,), (5, 3), (2, 3, 3), (1, 1, 5, 1)])
def test_axes(sections):
    T, H, D, R = 37, 3, 32, 16
    x, f = _x((T, H, D), torch.float32), _freq(R, 500.0, torch.float64)
    pos = torch.randint(-50, 1000, (len(sections), T),
                        generator=torch.Generator().manual_seed(2)).to(torch.int32).to(DEV)
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    angle = torch.stack([pos[a].double() * f[i] for i, a in enumerate(axis)], -1)
    want, size = rotate(x, angle[:, None])
    got = rotary(x, pos, f, sections=sections)
    assert_within(got, want, rotary_tolerance(want, size, x.dtype))
    # the same rows as [B, H, S, D] with positions per batch entry
    xb = x.permute(1, 0, 2)[None].expand(2, -1, -1, -1)
    gb = rotary(xb, pos[:, None].expand(-1, 2, -1), f, sections=sections)
    assert torch.equal(gb[0].permute(1, 0, 2), got) and torch.equal(gb[1], gb[0])


@pytest.mark.parametrize("far", [1 << 20, 1 << 24, 1 << 31, (1 << 40) + 12345])
def test_far_positions(far):
    """The angle keeps its precision: fp64 holds position * inv_freq within 2^-52 of itself, so
    at 2^40 radians the reference and the kernel may differ by 2 * 2^-52 * 2^40 = 2^-11."""
    x, f = _x((64, 2, 32), torch.float32), _freq(32)
    pos = torch.arange(far, far + 64, device=DEV)
    want, size = rotate(x, (pos.double()[:, None] * f.double())[:, None])
    tol = rotary_tolerance(want, size, x.dtype) + size * 4 * far * 2.0 ** -52
    assert_within(rotary(x, pos, f), want, tol)


def test_strides_in_place_and_gradient():
    big = _x((2, 9, 4, 3 * 64), torch.bfloat16)                # [B, S, H, 3 D]
    x = big[..., 64:128].permute(0, 2, 1, 3)
    f, pos = _freq(64), torch.arange(9, dtype=torch.int32, device=DEV)
    want = rotary(x.contiguous(), pos, f)
    kept = big.clone()
    assert torch.equal(rotary(x, pos, f), want)
    assert rotary(x, pos, f, out=x) is x and torch.equal(x, want)
    assert torch.equal(big[..., :64], kept[..., :64]) and torch.equal(big[..., 128:], kept[..., 128:])
    # the inverse is the transpose: <rotary(x), y> = <x, inverse(y)>, and a difference quotient
    a, y = _x((5, 2, 64), torch.float32, 3), _x((5, 2, 64), torch.float32, 4)
    p = torch.arange(5, device=DEV) * 17
    grad = rotary(y, p, f, inverse=True).double()
    step = _x((5, 2, 64), torch.float32, 5)
    ahead, behind = rotary(a + 0.5 * step, p, f).double(), rotary(a - 0.5 * step, p, f).double()
    quotient = ((ahead - behind) * y.double()).sum()
    # 640 values of at most 2^3 and fp32 operands: rounding 640 * 2^6 * 2^-22
    assert abs(float(quotient - (grad * step.double()).sum())) < 640 * 64 * 2.0 ** -22


def test_streams_graph_and_empty():
    x, f = _x((33, 4, 128), torch.float16), _freq(128)
    pos = torch.arange(33, dtype=torch.int32, device=DEV)
    want = rotary(x, pos, f)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.empty_like(x)
    with torch.cuda.stream(side):
        rotary(x, pos, f, out=out)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        rotary(x, pos, f, out=out)
    pos.add_(5)
    graph.replay()
    assert torch.equal(out, rotary(x, pos, f))
    assert rotary(x[:0], pos[:0], f).shape == (0, 4, 128)
    assert rotary(x[:, :0], pos, f).shape == (33, 0, 128)


def test_refusals_of_the_library():
    x, pos = _x((4, 2, 64), torch.bfloat16), torch.arange(4, device=DEV)
    with pytest.raises(FaError, match="head dim"):
        rotary(x, pos, _freq(24))                              # R = 24
    with pytest.raises(FaError, match="head dim"):
        rotary(x, pos, _freq(80))                              # R > D
    with pytest.raises(FaError, match="align"):
        rotary(_x((4, 2, 68), torch.bfloat16)[..., :64], pos, _freq(64))


def test_out_of_memory_keeps_its_type():
    """A broadcast input may ask for an output that no device holds (2^40 values)."""
    x, pos = _x((1, 1, 64), torch.bfloat16), torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises(torch.OutOfMemoryError):
        rotary(x.expand(1 << 28, 64, 64), pos.expand(1 << 28), _freq(64))
    y = _x((4, 2, 64), torch.bfloat16)
    assert torch.equal(rotary(y, pos.expand(4), _freq(64)), y)     # angle 0: x


@pytest.mark.parametrize("B,H,S,D,R", [(1, 4096, 2, 256, 256), (1, 2, 5000, 64, 32),
                                       (3, 7, 1999, 128, 128), (1, 65536, 1, 16, 16)])
def test_wide_rows_and_many(B, H, S, D, R):
    """Rows of more items than a CTA takes at once, and more rows than one wave of CTAs."""
    x, f = _x((B, H, S, D), torch.bfloat16), _freq(R)
    pos = torch.arange(S, device=DEV) * 3
    want, size = rotate(x, pos.double()[:, None] * f.double())
    assert_within(rotary(x, pos, f), want, rotary_tolerance(want, size, x.dtype))
