"""paged_kv_append and paged_attention against their definitions in fp64: head
groups, head dims, page sizes, ragged and empty sequences, masks, strides,
streams, graphs, pages outside the cache."""

import pytest
import torch

from cs348k_fast_attention_grammar_b200 import (attention, device_status, paged_attention,
                                                paged_kv_append)
from paged_reference import (Cache, assert_within, attention as reference, attention_tolerance,
                             borders, rotary_tolerance, rotate)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FA_ERR_PAGE = 14
BF16, F16 = torch.bfloat16, torch.float16


def _randn(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


# Which kernel runs, and how its work is cut, goes by the keys that the table has room for: the
# sequences' own, 8192, 2^18.
ROOMS = (0, 8192, 1 << 18)


def _with_room(table, page, keys):
    """The table with entries (outside the cache) for that many keys."""
    more = -(-keys // page) - table.shape[1]
    return table if more <= 0 else torch.nn.functional.pad(table, (0, more), value=-3)


def _check(q_lens, kv_lens, Hq, Hkv, D, page, dtype=BF16, causal=True, hnd=False, seed=0,
           scale=None, **kw):
    c = Cache(kv_lens, page, Hkv, D, dtype, DEV, seed=seed, hnd=hnd)
    q = _randn((sum(q_lens), Hq, D), dtype, seed + 1)
    cu = borders(q_lens, DEV)
    want, size = reference(q, c.k, c.v, c.table, kv_lens, q_lens, causal, scale)
    tol = attention_tolerance(want, size, dtype, max(kv_lens))
    kw.setdefault("max_q_len", max(q_lens))
    for room in ROOMS:
        table = _with_room(c.table, page, room)
        out = torch.full_like(q, float("nan"))
        got = paged_attention(q, c.k, c.v, table, c.lens, cu_seqlens=cu, causal=causal,
                              scale=scale, out=out, **kw)
        assert_within(got, want, tol, f"{q_lens} over {kv_lens}, room for {room}")
        assert device_status() == 0
    return q, c, cu, got


# --------------------------------------------------------------------------- single tokens
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (4, 4), (8, 2), (6, 2), (5, 1), (16, 1), (48, 2),
                                    (128, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_single_tokens_heads(dtype, Hq, Hkv, D):
    _check([1, 1, 1], [1, 77, 300], Hq, Hkv, D, 16, dtype)


@pytest.mark.parametrize("D", [8, 16, 40, 72, 80, 96, 120])
def test_head_dims(D):
    _check([1, 3, 1], [64, 130, 31], 4, 2, D, 32)
    _check([70, 3], [64 + 70, 130], 8, 2, D, 32)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
def test_page_sizes(page):
    lens = [page - 1, page, page + 1, 3 * page + 7]
    _check([1] * 4, lens, 8, 2, 64, page)
    _check([min(n, 9) for n in lens], lens, 8, 2, 128, page)
    _check([min(n, 140) for n in lens], lens, 8, 2, 128, page)


def test_every_length():
    """Lengths 0 to 130: every place a length can end in a page, a step and a block."""
    lens = list(range(0, 131))
    _check([1] * len(lens), lens, 4, 2, 64, 16)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hkv", [1, 2, 8, 24])
def test_clusters(D, Hkv):
    """One to eight CTAs over a sequence's keys, and lengths that leave some of them without."""
    for top in (700, 2500, 5000, 12000):
        _check([1, 3], [top, 17], 4 * Hkv, Hkv, D, 32)
        _check([0, 5], [top, top // 3], 2 * Hkv, Hkv, D, 64, F16, causal=False)


def test_long_and_many():
    _check([1, 1], [20000, 4097], 8, 1, 128, 64)
    _check([1] * 300, [(37 * i) % 500 for i in range(300)], 4, 2, 64, 16)
    _check([1, 0, 2] * 60, [100, 50, 333] * 60, 8, 8, 128, 32)


# --------------------------------------------------------------------------- chunks
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q_lens,kv_lens", [([2], [2]), ([7, 1, 0, 33], [7, 50, 90, 160]),
                                            ([127], [127]), ([128], [300]), ([129, 1], [129, 1]),
                                            ([300, 5], [300, 1029]), ([64, 65, 63], [64, 200, 129])])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (6, 2)])
def test_chunks(causal, D, q_lens, kv_lens, Hq, Hkv):
    _check(q_lens, kv_lens, Hq, Hkv, D, 16, causal=causal)


@pytest.mark.parametrize("g", [1, 3, 7, 16, 33, 100, 128])
def test_chunk_groups(g):
    _check([40, 1, 11], [100, 260, 11], g, 1, 64, 32, F16)
    _check([40, 1, 11], [100, 260, 11], 2 * g, 2, 128, 64)


def test_chunk_over_long_cache():
    _check([96], [9000], 16, 2, 128, 64)
    _check([300, 17], [3000, 8191], 8, 1, 128, 16, F16, causal=False)


@pytest.mark.parametrize("causal", [True, False])
def test_units_that_fill_the_device(causal):
    """640 and more units of 256 rows: none is split."""
    _check([300, 40, 520, 0, 1, 290], [300, 200, 520, 7, 90, 811], 64, 64, 64, 16, causal=causal)
    _check([300, 1100], [300, 1300], 128, 64, 128, 64, F16, causal=causal)


def test_long_units_among_many():
    """720 and more units, the longest of them beyond a CTA's even share of the key blocks: those
    are cut, the others are not."""
    _check([40] + [1] * 89, [6000] + [100 - i for i in range(89)], 8, 8, 64, 16)
    _check([3, 200, 9] + [1] * 250, [900, 7000, 5000] + [50] * 250, 8, 4, 128, 16, F16)
    _check([40] * 100, [4000] + [40] * 98 + [9000], 8, 8, 64, 32, causal=False)


@pytest.mark.parametrize("q_lens,kv_lens", [([520], [9000]), ([64, 700], [20000, 6000]),
                                            ([300] * 3, [4100, 4096, 300]), ([33], [33000])])
def test_units_cut_over_the_device(q_lens, kv_lens):
    _check(q_lens, kv_lens, 8, 2, 128, 64)
    _check(q_lens, kv_lens, 2, 1, 64, 32, F16, causal=False)


def test_rows_that_see_nothing():
    """kv_lens below the number of new tokens (0 among them): the tokens before the start see
    no key under the causal mask and get zeros."""
    _, _, _, got = _check([3, 5, 200, 1, 180], [0, 2, 0, 0, 30], 4, 2, 64, 16)
    assert not got[:3].any() and not got[3:6].any() and not got[8:208].any()
    assert not got[209:209 + 150].any() and got[209 + 150:].any()
    _check([3, 5, 200], [0, 2, 0], 4, 2, 128, 16, causal=False)


def test_hint_never_changes_what_is_computed():
    q_lens, kv_lens = [1, 90, 3, 20], [70, 500, 3, 1000]
    for hint in (None, 0, 1, 4, 90, 10 ** 6):
        _check(q_lens, kv_lens, 8, 2, 128, 32, max_q_len=hint)


def test_scale_and_score_jump():
    _check([1, 40], [100, 90], 4, 2, 64, 16, scale=0.0)
    # negative scales turn the order of the keys round
    _check([1, 40], [100, 90], 4, 2, 64, 16, scale=-0.2)
    for dtype in (BF16, F16):
        for q_lens in ([1], [150]):
            c = Cache([700], 64, 1, 64, dtype, DEV)
            q = _randn((q_lens[0], 2, 64), dtype, 3)
            page, row = int(c.table[0, 550 // 64]), 550 % 64
            c.k[page, row, 0] = q[0, 0] * 8
            want, size = reference(q, c.k, c.v, c.table, [700], q_lens)
            # scores reach 64 here instead of 8: the score term of the tolerance is 8 times larger
            tol = attention_tolerance(want, size, dtype, 700) + size * 7 * 2.0 ** -12.5
            for room in ROOMS:
                got = paged_attention(q, c.k, c.v, _with_room(c.table, 64, room), c.lens,
                                      cu_seqlens=borders(q_lens, DEV))
                assert_within(got, want, tol)


@pytest.mark.parametrize("room", ROOMS)
def test_non_finite_rows(room):
    """A query that is not a number makes its own outputs so and no others; a key that is not, or
    is infinite, the outputs of the tokens that see it."""
    q_lens, kv_lens = [1, 60, 40], [300, 60, 90]
    c = Cache(kv_lens, 16, 1, 64, BF16, DEV)
    table = _with_room(c.table, 16, room)
    cu = borders(q_lens, DEV)
    q = _randn((101, 2, 64), BF16, 1)
    want, size = reference(q, c.k, c.v, c.table, kv_lens, q_lens)
    tol = attention_tolerance(want, size, BF16, 300)
    q[7, 1] = float("nan")
    c.k[int(c.table[2, 70 // 16]), 70 % 16] = float("nan")     # seen by the last 20 tokens
    got = paged_attention(q, c.k, c.v, table, c.lens, cu_seqlens=cu, max_q_len=60)
    bad = torch.zeros((101, 2), dtype=torch.bool, device=DEV)
    bad[7, 1] = bad[81:, 0] = bad[81:, 1] = True
    assert got[bad].isnan().all()
    assert_within(got[~bad], want[~bad], tol[~bad])


def test_layouts_and_padded_rows():
    """A [pages, Hkv, page, D] allocation, q inside a fused projection, out inside a wider
    buffer, rows before and behind the sequences."""
    q_lens, kv_lens = [1, 140, 6], [33, 200, 6]
    for D, page, room in ((64, 16, 0), (128, 64, 0), (64, 16, 1 << 18), (128, 64, 1 << 18)):
        c = Cache(kv_lens, page, 2, D, BF16, DEV, hnd=True)
        rows = _randn((3 + sum(q_lens) + 5, 12 * D), BF16, 1)
        q = rows[:, 2 * D:10 * D].unflatten(1, (8, D))
        wide = torch.full((q.shape[0], 9, D + 8), 7.0, dtype=BF16, device=DEV)
        out = wide[:, 1:, :D]
        cu = borders(q_lens, DEV, first=3)
        table = _with_room(c.table, page, room)
        assert paged_attention(q, c.k, c.v, table, c.lens, cu_seqlens=cu, out=out) is out
        want, size = reference(q[3:-5], c.k, c.v, c.table, kv_lens, q_lens)
        assert_within(out[3:-5], want, attention_tolerance(want, size, BF16, 200))
        assert (wide[:3] == 7).all() and (wide[-5:] == 7).all()
        assert (wide[:, 0] == 7).all() and (wide[..., D:] == 7).all()
    assert device_status() == 0


def test_shared_pages():
    """Two sequences that share a prefix's pages, and a page that a sequence has twice."""
    c = Cache([96, 96], 32, 2, 64, BF16, DEV)
    c.table[1, :2] = c.table[0, :2]
    c.table[1, 2] = c.table[0, 0]
    q = _randn((2, 4, 64), BF16, 2)
    got = paged_attention(q, c.k, c.v, c.table, c.lens)
    want, size = reference(q, c.k, c.v, c.table, [96, 96], [1, 1])
    assert_within(got, want, attention_tolerance(want, size, BF16, 96))


def test_equals_attention_on_a_whole_prompt():
    """A prompt through the cache against the dense operator: both within the tolerance of the
    definition, so within twice of each other."""
    B, H, S, D = 2, 4, 333, 128
    q, k, v = (_randn((B, H, S, D), BF16, i) for i in range(3))
    page = 16
    n = -(-S // page)
    table = torch.randperm(B * n, generator=torch.Generator().manual_seed(0)).to(torch.int32)
    table = table.view(B, n).to(DEV)
    kc, vc = (torch.zeros((B * n, page, H, D), dtype=BF16, device=DEV) for _ in range(2))
    pack = lambda t: t.permute(0, 2, 1, 3).reshape(B * S, H, D)  # noqa: E731
    lens = torch.full((B,), S, dtype=torch.int32, device=DEV)
    cu = borders([S] * B, DEV)
    assert paged_kv_append(pack(k), pack(v), kc, vc, table, lens, cu_seqlens=cu) is None
    got = paged_attention(pack(q), kc, vc, table, lens, cu_seqlens=cu)
    dense = pack(attention(q, k, v, causal=True))
    want, size = reference(pack(q), kc, vc, table, [S] * B, [S] * B)
    tol = attention_tolerance(want, size, BF16, S)
    assert_within(got, want, tol)
    assert_within(got, dense.double(), 2 * tol)


def test_repeatable():
    for q_lens, kv_lens in (([1, 1], [9000, 300]), ([200, 1], [5000, 300]), ([900] * 9, [3000] * 9)):
        for room in ROOMS:
            q, c, cu, _ = _check(q_lens, kv_lens, 8, 2, 128, 64)
            table = _with_room(c.table, 64, room)
            made = [paged_attention(q, c.k, c.v, table, c.lens, cu_seqlens=cu,
                                    max_q_len=max(q_lens)) for _ in range(4)]
            assert all(torch.equal(m, made[0]) for m in made)


# --------------------------------------------------------------------------- far places
def test_cache_beyond_32_bit_offsets():
    """Caches of 2^31 + elements each; the sequence's pages are the last ones."""
    page, Hkv, D = 64, 8, 128
    pages = (1 << 31) // (page * Hkv * D) + 40
    kc, vc = (torch.empty((pages, page, Hkv, D), dtype=BF16, device=DEV) for _ in range(2))
    small = Cache([1500, 130], page, Hkv, D, BF16, DEV)
    shift = pages - small.pages
    kc[shift:], vc[shift:] = small.k, small.v
    table = torch.where(small.table >= 0, small.table + shift, small.table)
    k, v = _randn((2, Hkv, D), BF16, 1), _randn((2, Hkv, D), BF16, 2)
    paged_kv_append(k, v, kc, vc, table, small.lens)
    paged_kv_append(k, v, small.k, small.v, small.table, small.lens)
    assert torch.equal(kc[shift:].nan_to_num(5), small.k.nan_to_num(5))
    assert torch.equal(vc[shift:].nan_to_num(5), small.v.nan_to_num(5))
    for q_lens in ([1, 1], [200, 1]):
        for room in ROOMS:
            q = _randn((sum(q_lens), 16, D), BF16, 3)
            cu = borders(q_lens, DEV)
            a = paged_attention(q, kc, vc, _with_room(table, page, room), small.lens,
                                cu_seqlens=cu)
            assert torch.equal(a, paged_attention(q, small.k, small.v,
                                                  _with_room(small.table, page, room), small.lens,
                                                  cu_seqlens=cu))
    assert device_status() == 0


# --------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,Hkv,D,R,page,axes,interleaved", [
    (4, 2, 64, 64, 16, 1, False), (8, 8, 128, 64, 64, 1, True), (3, 1, 80, 32, 32, 3, False),
    (0, 2, 128, 128, 16, 1, False), (2, 2, 24, 16, 16, 2, True), (40, 8, 128, 128, 128, 3, False)])
def test_append(dtype, Hq, Hkv, D, R, page, axes, interleaved):
    q_lens, kv_lens = [5, 0, 1, 70, 3], [5, 40, 17, 200, 2]     # the last: one token too many
    T = sum(q_lens) + 4
    c = Cache(kv_lens, page, Hkv, D, dtype, DEV, hnd=(D == 128))
    kc, vc = c.k.clone(), c.v.clone()
    rows = _randn((T, (Hq + 2 * Hkv) * D), dtype, 1)
    q, k, v = (t.unflatten(1, (-1, D)) if t.shape[1] else None
               for t in rows.split([Hq * D, Hkv * D, Hkv * D], 1))
    f = (10000.0 ** (-torch.arange(0, R, 2) / R)).to(DEV)
    cu = borders(q_lens, DEV, first=2)
    place = torch.tensor([kv - n + i for n, kv in zip(q_lens, kv_lens) for i in range(n)])
    sections = positions = None
    if axes == 1:
        pos = place.to(DEV)
        angle = pos.double()[:, None] * f.double()
    else:
        sections = (R // 2 - (axes - 1) * 2,) + (2,) * (axes - 1)
        positions = torch.randint(0, 900, (axes, T), device=DEV)
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
        angle = torch.stack([positions[a, 2:-2].double() * f[i] for i, a in enumerate(axis)], -1)
    out = None if q is None else torch.full_like(q, 3.0)
    got = paged_kv_append(k, v, c.k, c.v, c.table, c.lens, cu_seqlens=cu, q=q, q_out=out,
                          inv_freq=f, positions=positions, sections=sections,
                          interleaved=interleaved)
    assert got is out
    if q is not None:
        want, size = rotate(q[2:-2], angle[:, None], interleaved)
        assert_within(out[2:-2], want, rotary_tolerance(want, size, dtype), "q")
        assert (out[:2] == 3).all() and (out[-2:] == 3).all()
    want, size = rotate(k[2:-2], angle[:, None], interleaved)
    tol = rotary_tolerance(want, size, dtype)
    row = 0
    for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        for i in range(n):
            at = kv - n + i
            if at >= 0:
                pg, r = int(c.table[b, at // page]), at % page
                assert_within(c.k[pg, r], want[row], tol[row], f"k {b} {i}")
                assert torch.equal(c.v[pg, r], v[2 + row])
                c.k[pg, r], c.v[pg, r] = kc[pg, r], vc[pg, r]
            row += 1
    # nothing else was written
    assert torch.equal(c.k.nan_to_num(9), kc.nan_to_num(9))
    assert torch.equal(c.v.nan_to_num(9), vc.nan_to_num(9))
    assert device_status() == 0


def test_append_in_place_queries_and_single_tokens():
    c = Cache([1, 30, 64], 16, 2, 64, BF16, DEV)
    q, k, v = (_randn((3, h, 64), BF16, h) for h in (4, 2, 3))
    v = v[:, :2]
    f = (10000.0 ** (-torch.arange(0, 64, 2) / 64)).to(DEV)
    want = paged_kv_append(k, v, c.k, c.v, c.table, c.lens, q=q, inv_freq=f)
    again = paged_kv_append(k, v, c.k, c.v, c.table, c.lens, cu_seqlens=borders([1] * 3, DEV),
                            q=q, q_out=q, inv_freq=f)
    assert again is q and torch.equal(q, want)


def test_places_outside_the_cache():
    """Reported by the status word, nothing written or read outside; other sequences go on."""
    c = Cache([20, 40], 16, 1, 64, BF16, DEV, wider=0)
    k, v, q = (_randn((2, 1, 64), BF16, i) for i in range(3))
    good, kc, vc = c.table.clone(), c.k.clone(), c.v.clone()
    for bad in (-1, c.pages, 2 ** 31 - 1, -2 ** 31):
        c.table[0, 1] = bad
        paged_kv_append(k, v, c.k, c.v, c.table, c.lens)
        assert device_status() == FA_ERR_PAGE and device_status() == 0
        pg = int(good[1, 2])
        assert torch.equal(c.k[pg, 7], k[1]) and torch.equal(c.v[pg, 7], v[1])
        c.k[pg, 7], c.v[pg, 7] = kc[pg, 7], vc[pg, 7]
        assert torch.equal(c.k.nan_to_num(9), kc.nan_to_num(9))
        for q_lens in ([1, 1], [19, 40]):
            for room in ROOMS:
                qq = q.repeat(30, 1, 1)[:sum(q_lens)]
                got = paged_attention(qq, c.k, c.v, _with_room(c.table, 16, room), c.lens,
                                      cu_seqlens=borders(q_lens, DEV))
                assert device_status() == FA_ERR_PAGE
                want, size = reference(qq[q_lens[0]:], c.k, c.v, good[1:], [40], q_lens[1:])
                assert_within(got[q_lens[0]:], want, attention_tolerance(want, size, BF16, 40))
    c.table.copy_(good)
    # a length behind the table: 3 pages hold 48
    lens = torch.tensor([20, 60], dtype=torch.int32, device=DEV)
    paged_kv_append(k, v, c.k, c.v, c.table, lens)
    assert device_status() == FA_ERR_PAGE
    got = paged_attention(q, c.k, c.v, c.table, lens)
    assert device_status() == FA_ERR_PAGE and got[0].isfinite().all()
    # negative lengths are empty, not errors
    lens = torch.tensor([20, -5], dtype=torch.int32, device=DEV)
    assert not paged_attention(q, c.k, c.v, c.table, lens)[1].any()
    assert device_status() == 0


def test_borders_outside_the_rows():
    """Borders are held to the packed rows, whatever they hold."""
    c = Cache([20, 40], 16, 1, 64, BF16, DEV)
    q = _randn((4, 2, 64), BF16, 1)
    for cu in ([0, 1, 900], [-5, 1, 2], [3, 1, 2], [0, 2 ** 31 - 1, 1]):
        t = torch.tensor(cu, dtype=torch.int32, device=DEV)
        for room in ROOMS:
            table = _with_room(c.table, 16, room)
            for longest in (None, 1, 200):
                paged_attention(q, c.k, c.v, table, c.lens, cu_seqlens=t, max_q_len=longest)
        paged_kv_append(q[:, :1], q[:, :1], c.k.clone(), c.v.clone(), c.table, c.lens, cu_seqlens=t)
        torch.cuda.synchronize()
    device_status()


def test_empty_calls():
    c = Cache([20], 16, 2, 64, BF16, DEV)
    none = torch.zeros((0, 2, 64), dtype=BF16, device=DEV)
    cu = torch.zeros(2, dtype=torch.int32, device=DEV)
    assert paged_attention(none, c.k, c.v, c.table, c.lens, cu_seqlens=cu).shape == (0, 2, 64)
    assert paged_kv_append(none, none, c.k, c.v, c.table, c.lens, cu_seqlens=cu) is None
    # rows, but no sequence owns one
    q = _randn((3, 2, 64), BF16)
    for room in ROOMS:
        for longest in (1, 100):
            out = torch.full_like(q, 2.0)
            paged_attention(q, c.k, c.v, _with_room(c.table, 16, room), c.lens, cu_seqlens=cu,
                            max_q_len=longest, out=out)
            assert (out == 2).all()


# --------------------------------------------------------------------------- a user's program
def _steps(state, c, f):
    q, k, v, cu, longest = state
    r = paged_kv_append(k, v, c.k, c.v, c.table, c.lens, cu_seqlens=cu, q=q, inv_freq=f)
    return paged_attention(r, c.k, c.v, c.table, c.lens, cu_seqlens=cu, max_q_len=longest)


@pytest.mark.parametrize("D", [64, 128])
def test_generation_matches_one_prompt(D):
    """A prompt in chunks, then token by token, through append and attention: every row within
    the tolerance of the definition over the rotated keys that the cache then holds."""
    Hq, Hkv, page, total = 8, 2, 16, 150
    f = (10000.0 ** (-torch.arange(0, D, 2) / D)).to(DEV)
    rows = _randn((2, total, (Hq + 2 * Hkv), D), BF16)
    c = Cache([total, total], page, Hkv, D, BF16, DEV)
    c.k.fill_(float("nan"))
    c.v.fill_(float("nan"))
    for at, n in ((0, 70), (70, 33), (103, 45), (148, 1), (149, 1)):
        new = rows[:, at:at + n].flatten(0, 1)
        q, k, v = new.split([Hq, Hkv, Hkv], 1)
        c.lens.fill_(at + n)
        got = _steps((q, k, v, borders([n, n], DEV), n), c, f)
        pos = torch.arange(at, at + n, device=DEV).repeat(2)
        qr, _ = rotate(q, (pos.double()[:, None] * f.double())[:, None])
        want, size = reference(qr, c.k, c.v, c.table, [at + n] * 2, [n, n])
        # the queries' own rounding: half a step of each of D products, at most 2^-9 * sum |q k|
        # * scale <= 2^-9 * 128 * 0.64 / 11.3 in the exponent, twice over (weight and sum)
        tol = attention_tolerance(want, size, BF16, total) + size * 2 * 2.0 ** -9 * 7.3
        assert_within(got, want, tol, f"rows {at}..{at + n}")
    assert device_status() == 0


@pytest.mark.parametrize("room", ROOMS)
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [90, 1, 30]])
def test_graphs_with_new_lengths(q_lens, room):
    """Two captured steps with outputs of their own, replayed in two streams at once with lengths
    and tokens changed in place, against eager calls."""
    D, Hq, Hkv, page = 128, 8, 2, 16
    f = (10000.0 ** (-torch.arange(0, D, 2) / D)).to(DEV)
    sides = [torch.cuda.Stream() for _ in range(2)]
    made = []
    for i, side in enumerate(sides):
        c = Cache([2500, 300, 120], page, Hkv, D, BF16, DEV, seed=i)
        c.table = _with_room(c.table, page, room)
        T = sum(q_lens)
        q, k, v = (_randn((T, h, D), BF16, 10 * i + h) for h in (Hq, Hkv, Hkv))
        state = (q, k, v, borders(q_lens, DEV), max(q_lens))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _steps(state, c, f)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = _steps(state, c, f)
        made.append((c, state, graph, out, side))
    for lens in ([2500, 300, 120], [2000, 200, 100], [100, 290, 35]):
        for c, state, *_ in made:
            c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
            state[0].mul_(0.75)
        torch.cuda.synchronize()
        for _ in range(3):
            for _, _, graph, _, side in made:
                with torch.cuda.stream(side):
                    graph.replay()
        torch.cuda.synchronize()
        got = [out.clone() for _, _, _, out, _ in made]
        for (c, state, *_), o in zip(made, got):
            assert torch.equal(_steps(state, c, f), o)
    assert device_status() == 0


@pytest.mark.parametrize("room", ROOMS)
@pytest.mark.parametrize("q_lens", [[1, 1], [150, 1]])
def test_streams_at_once(q_lens, room):
    """Calls in two streams at once, each with its own inputs, against the calls alone."""
    cs = [Cache([3000, 200], 16, 2, 64, BF16, DEV, seed=i) for i in range(2)]
    qs = [_randn((sum(q_lens), 8, 64), BF16, i) for i in range(2)]
    cu = borders(q_lens, DEV)

    def call(q, c):
        return paged_attention(q, c.k, c.v, c.table, c.lens, cu_seqlens=cu, max_q_len=q_lens[0])

    for c in cs:
        c.table = _with_room(c.table, 16, room)
    want = [call(q, c) for q, c in zip(qs, cs)]
    sides = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[i].append(call(qs[i], cs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


@pytest.mark.parametrize("room", ROOMS)
@pytest.mark.parametrize("q_lens", [[1, 1], [150, 1]])
def test_handed_from_stream_to_stream(q_lens, room):
    """Keys stored in one stream and read in another, step by step through events."""
    c = Cache([3000, 200], 16, 2, 64, BF16, DEV)
    c.table = _with_room(c.table, 16, room)
    cu, f = borders(q_lens, DEV), torch.ones(32, device=DEV)
    n = sum(q_lens)
    steps = [(_randn((n, 8, 64), BF16, i), _randn((n, 2, 64), BF16, i + 50),
              _randn((n, 2, 64), BF16, i + 90)) for i in range(10)]
    r = torch.empty_like(steps[0][0])

    def store(q, k, v):
        paged_kv_append(k, v, c.k, c.v, c.table, c.lens, cu_seqlens=cu, q=q, inv_freq=f, q_out=r)

    def read(out=None):
        return paged_attention(r, c.k, c.v, c.table, c.lens, cu_seqlens=cu, max_q_len=q_lens[0],
                               out=out)

    want = []
    for step in steps:
        store(*step)
        want.append(read())
    got = [torch.empty_like(o) for o in want]
    left, right = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for step, out in zip(steps, got):
        left.wait_stream(right)
        with torch.cuda.stream(left):
            store(*step)
        right.wait_stream(left)
        with torch.cuda.stream(right):
            read(out)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
