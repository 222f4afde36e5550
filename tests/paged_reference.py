"""fp64 forms of the rotary and paged operators, and their tests' tolerances."""

import math

import torch


def half_step(dtype):
    """A rounding to nearest is off by at most this, relative to the value."""
    return torch.finfo(dtype).eps / 2


def rotate(x, angle, interleaved=False, inverse=False):
    """x [..., D] by angle [..., R/2]: (fp64 result, sum of magnitudes of each value's terms)."""
    x = x.double()
    angle = -angle if inverse else angle
    R = 2 * angle.shape[-1]
    y, size = x.clone(), torch.zeros_like(x)
    ia = torch.arange(0, R, 2) if interleaved else torch.arange(R // 2)
    ib = ia + (1 if interleaved else R // 2)
    ia, ib = ia.to(x.device), ib.to(x.device)
    a, b = x[..., ia], x[..., ib]
    y[..., ia] = a * angle.cos() - b * angle.sin()
    y[..., ib] = b * angle.cos() + a * angle.sin()
    size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return y, size


def rotary_tolerance(y, size, dtype):
    """The angle's remainder is rounded once to fp32 (2^-24 of half a turn, 2^-22.3
    in radians), sine and cosine are within 2^-23, and the two products and their
    sum add 2 * 2^-24: together below 2^-21 of |a| + |b|.  Then one rounding to
    the output's type (fp16 results below 2^-14: 2^-25)."""
    return size * 2.0 ** -21 + (y.abs() + size * 2.0 ** -21) * half_step(dtype) + 2.0 ** -25


def attention(q, k_cache, v_cache, table, kv_lens, q_lens, causal=True, scale=None, starts=None):
    """Packed fp64 output and, per value, sum_j p_j |v_j| (rows of no sequence: nan)."""
    T, Hq, D = q.shape
    page, Hkv = k_cache.shape[1], k_cache.shape[2]
    g = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.full((T, Hq, D), float("nan"), dtype=torch.float64, device=q.device)
    size = out.clone()
    row = 0
    for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        if starts is not None:
            row = starts[b]
        if n == 0:
            continue
        ids = table[b, :-(-kv // page)].long()
        k = k_cache[ids].flatten(0, 1)[:kv].double()
        v = v_cache[ids].flatten(0, 1)[:kv].double()
        place = torch.arange(kv - n, kv, device=q.device)[:, None]
        seen = torch.ones((n, kv), dtype=torch.bool, device=q.device)
        if causal:
            seen = torch.arange(kv, device=q.device)[None] <= place
        for h in range(Hkv):
            qh = q[row:row + n, h * g:(h + 1) * g].double()
            s = torch.einsum("nge,ke->gnk", qh, k[:, h]) * scale
            s = s.masked_fill(~seen, -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)       # a row that sees nothing: zeros
            out[row:row + n, h * g:(h + 1) * g] = torch.einsum("gnk,ke->nge", p, v[:, h])
            size[row:row + n, h * g:(h + 1) * g] = torch.einsum("gnk,ke->nge", p, v[:, h].abs())
        row += n
    return out, size


def attention_tolerance(out, size, dtype, keys):
    """Each weight is rounded to the 16-bit type (half a step of it; fp16 weights
    below 2^-14 of the row's reference: 2^-25 each).  Scores are fp32 sums of D
    <= 128 exact products of unit normals: 128 * 2^-23 * scale * sum |q k| is at
    most 2^-12.5 in the exponent, an exponential is within 2^-13.7, and sums of
    the weights within 2^-13: together below 2^-11.  Then the output's rounding."""
    weights = half_step(dtype) + 2.0 ** -11
    rare = keys * 2.0 ** -25 if dtype == torch.float16 else 0.0
    near = size * weights + rare
    return near + (out.abs() + near) * half_step(dtype) + 2.0 ** -25


def assert_within(got, want, tol, what=""):
    bad = (got.double() - want).abs() > tol
    bad |= got.double().isnan() & ~want.isnan()
    if bool(bad.any()):
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off, first at {at}: "
                             f"{got[at].item()} for {want[at].item()}, tolerance {tol[at].item()}")


class Cache:
    """A paged batch: NaN in every slot that no sequence owns, pages in random order."""

    def __init__(self, kv_lens, page, Hkv, D, dtype, device, seed=0, spare=3, hnd=False,
                 amplitude=1.0, wider=2):
        gen = torch.Generator().manual_seed(seed)
        used = [-(-kv // page) for kv in kv_lens]
        self.pages = sum(used) + spare
        order = torch.randperm(self.pages, generator=gen).tolist()
        width = max(used + [1]) + wider
        table = torch.full((len(kv_lens), width), -7, dtype=torch.int32)
        shape = ((self.pages, Hkv, page, D) if hnd else (self.pages, page, Hkv, D))
        self.k, self.v = (torch.full(shape, float("nan"), dtype=dtype) for _ in range(2))
        if hnd:
            self.k, self.v = self.k.permute(0, 2, 1, 3), self.v.permute(0, 2, 1, 3)
        for b, (n, kv) in enumerate(zip(used, kv_lens)):
            for i in range(n):
                pg = order.pop()
                table[b, i] = pg
                rows = min(page, kv - i * page)
                for c in (self.k, self.v):
                    c[pg, :rows] = (torch.randn((rows, Hkv, D), generator=gen)
                                    * amplitude).to(dtype)
        strides = self.k.stride()
        self.k, self.v, self.table = (t.to(device) for t in (self.k, self.v, table))
        assert self.k.stride() == strides
        self.lens = torch.tensor(kv_lens, dtype=torch.int32, device=device)


def borders(q_lens, device, first=0):
    out = [first]
    for n in q_lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=device)
