"""Edges of the paged operators against their definitions in fp64: infinite scores, weights of
masked keys, scales near zero, lengths and pages that the table does not hold, borders outside the
packed rows, the order of what the status word reports."""

import math

import pytest
import torch

from cs348k_fast_attention_grammar_b200 import (_lib, device_status, paged_attention,
                                                paged_kv_append)
from paged_reference import (Cache, assert_within, attention as reference, attention_tolerance,
                             borders)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FA_ERR_TIMEOUT, FA_ERR_PAGE = 11, 14
BF16, F16 = torch.bfloat16, torch.float16
INF = float("inf")

# (tokens, lengths, query heads, key heads, room in the table): clusters of the row kernel, its whole
# units, its split ranges; the tile kernel with whole units and with cut ones.
PATHS = {
    "clusters": ([1, 60, 40], [300, 60, 90], 2, 1, 0),
    "whole": ([3, 16, 9] * 40, [300, 60, 90] * 40, 8, 4, 0),
    "split": ([3, 16, 9], [300, 60, 90], 2, 1, 1 << 18),
    "tiles": ([1, 60, 40], [300, 60, 90], 8, 4, 1 << 18),
    "tiles cut": ([200, 3], [5000, 700], 8, 2, 1 << 18),
}


def _randn(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


def _problem(path, dtype=BF16, D=64, page=16):
    q_lens, kv_lens, Hq, Hkv, room = PATHS[path]
    c = Cache(kv_lens, page, Hkv, D, dtype, DEV)
    more = max(0, -(-room // page) - c.table.shape[1])
    c.table = torch.nn.functional.pad(c.table, (0, more), value=-3)
    q = _randn((sum(q_lens), Hq, D), dtype, 1)
    return c, q, q_lens, kv_lens


def _call(c, q, q_lens, **kw):
    return paged_attention(q, c.k, c.v, c.table, c.lens, cu_seqlens=borders(q_lens, DEV),
                           max_q_len=max(q_lens), **kw)


def _slot(c, b, key):
    page = c.k.shape[1]
    return int(c.table[b, key // page]), key % page


def _definition(c, q, q_lens, kv_lens):
    """Causal attention in fp64 as it is written, and sum_j p_j |v_j|: a score of +inf or NaN makes
    its row NaN, one of -inf has no weight, a row all of whose scores are -inf is zero."""
    scale = 1.0 / math.sqrt(q.shape[2])
    out, size, g, row = [], [], q.shape[1] // c.k.shape[2], 0
    for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        ids = c.table[b, :-(-kv // c.k.shape[1])].long()
        k, v = (t[ids].flatten(0, 1)[:kv].double().repeat_interleave(g, 1) for t in (c.k, c.v))
        # (products and their sum one by one: a matrix product may order infinities otherwise)
        s = (q[row:row + n, None].double() * k[None]).sum(-1).movedim(2, 1) * scale
        hidden = torch.arange(kv, device=DEV) > torch.arange(kv - n, kv, device=DEV)[:, None]
        s = s.masked_fill(hidden[:, None], -INF)
        p = torch.softmax(s, -1)
        p = torch.where((s == -INF).all(-1, keepdim=True), 0.0, p)
        out.append(torch.einsum("nhk,khe->nhe", p, v))
        size.append(torch.einsum("nhk,khe->nhe", p, v.abs()))
        row += n
    return torch.cat(out), torch.cat(size)


# --------------------------------------------------------------------------- infinite scores
def _assert_nan_alike(got, want, tol, what):
    bad = want.isnan()
    assert torch.equal(got.isnan(), bad), f"{what}: {int((got.isnan() != bad).sum())} values"
    assert_within(got[~bad], want[~bad], tol[~bad], what)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("path", PATHS)
def test_infinite_keys(path, dtype):
    """One infinite channel of one key, at every place of 16: a token that sees it gets NaN where
    its score is +inf, and no weight of it where the score is -inf."""
    for place in range(16):
        c, q, q_lens, kv_lens = _problem(path, dtype)
        b = q_lens.index(max(q_lens))
        key = kv_lens[b] - 16 + place
        pg, r = _slot(c, b, key)
        c.k[pg, r, 0, 3] = INF if place % 4 < 2 else -INF
        q[sum(q_lens[:b + 1]) - 1, 0, 3] = 1 if place % 4 < 2 else -1
        want, size = _definition(c, q, q_lens, kv_lens)
        tol = attention_tolerance(want, size, dtype, max(kv_lens))
        assert want.isnan().any() and not want.isnan().all()
        _assert_nan_alike(_call(c, q, q_lens), want, tol, f"{path}, key {key}")
    assert device_status() == 0


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("path", PATHS)
def test_infinite_queries(path, dtype):
    """One infinite channel of a query: its row is NaN if a key that it sees has that channel on
    the same side of zero."""
    c, q, q_lens, kv_lens = _problem(path, dtype)
    at = torch.arange(q.shape[0], device=DEV) % 3 == 1
    q[at, :, 5] = INF
    want, size = _definition(c, q, q_lens, kv_lens)
    tol = attention_tolerance(want, size, dtype, max(kv_lens))
    assert want.isnan().any()
    _assert_nan_alike(_call(c, q, q_lens), want, tol, path)


def test_an_infinite_score_of_rows_that_see_few_keys():
    """A prompt whose tokens see 1, 2, 3, ... keys, each key's score +inf in turn."""
    n = 40
    for Hkv, room in ((1, 0), (8, 1 << 18)):
        for place in range(16):
            c = Cache([n], 16, Hkv, 64, BF16, DEV)
            c.table = torch.nn.functional.pad(c.table, (0, room // 16), value=-3)
            q = _randn((n, 2 * Hkv, 64), BF16, 2)
            q[:, :, 9] = 1
            pg, r = _slot(c, 0, place)
            c.k[pg, r, :, 9] = INF
            got = _call(c, q, [n])
            assert got[place:].isnan().all(), (Hkv, place)
            assert got[:place].isfinite().all(), (Hkv, place)


# --------------------------------------------------------------------------- masked keys
@pytest.mark.parametrize("path", PATHS)
def test_masked_keys_have_no_weight(path):
    """Tokens that see values of zero get zeros, whatever finite values the later ones hold."""
    c, q, q_lens, kv_lens = _problem(path)
    row = 0
    for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        ids = c.table[b, :-(-kv // 16)].long()
        v = c.v[ids].flatten(0, 1)
        v[:kv] = 0
        v[kv - n // 2:kv] = 2.0 ** 110
        c.v[ids] = v.unflatten(0, (len(ids), 16))
    want, size = reference(q, c.k, c.v, c.table, kv_lens, q_lens)
    got = _call(c, q, q_lens)
    assert_within(got, want, attention_tolerance(want, size, BF16, max(kv_lens)), path)
    for n in q_lens:
        assert not got[row:row + n - n // 2].any(), f"{path}, rows {row}.."
        row += n


# --------------------------------------------------------------------------- scales
@pytest.mark.parametrize("path", PATHS)
def test_scales_near_zero(path):
    """Scores of 10^35 under a scale of 10^-36, and no scale at all."""
    c, q, q_lens, kv_lens = _problem(path)
    want, size = reference(q, c.k, c.v, c.table, kv_lens, q_lens)
    tol = attention_tolerance(want, size, BF16, max(kv_lens))
    # powers of two change no rounding: (2^57 q) (2^60 k) 2^-120 = q k / 8
    big_q, kept = q * 2.0 ** 57, c.k.clone()
    c.k.mul_(2.0 ** 60)
    assert_within(_call(c, big_q, q_lens, scale=2.0 ** -120), want, tol, path)
    c.k.copy_(kept)
    # a scale of zero weighs all keys alike, and an infinite score is no number then
    want, size = reference(q, c.k, c.v, c.table, kv_lens, q_lens, True, 0.0)
    assert_within(_call(c, q, q_lens, scale=0.0), want,
                  attention_tolerance(want, size, BF16, max(kv_lens)), path)
    pg, r = _slot(c, 0, kv_lens[0] - 1)
    c.k[pg, r, :, 7] = -INF
    last = q_lens[0] - 1
    q[last, :, 7] = 1
    got = _call(c, q, q_lens, scale=0.0)
    assert got[last].isnan().all() and got[:last].isfinite().all()


# --------------------------------------------------------------------------- outside the table
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_lens,Hkv,pages", [([1, 1], 2, 3), ([20, 9], 2, 3), ([100, 90], 8, 3),
                                              ([16, 9], 2, 3000), ([20, 16], 8, 400),
                                              ([100, 90], 8, 400),
                                              ([100, 90], 1, 400), ([300, 20], 1, 900)])
def test_lengths_beyond_the_table(q_lens, Hkv, pages, causal):
    """Tokens keep their places, which append stores them by; they see the keys that the table
    holds."""
    held = 16 * pages
    beyond = 12
    kv_lens = [held, held - 5]
    c = Cache(kv_lens, 16, Hkv, 64, BF16, DEV, wider=0)
    q = _randn((sum(q_lens), 2 * Hkv, 64), BF16, 3)
    c.lens[0] += beyond
    got = _call(c, q, q_lens, causal=causal)
    assert device_status() == FA_ERR_PAGE
    # the first sequence again, with its table as long as its length (the keys there hidden below)
    n = q_lens[0]
    seen = torch.arange(held, device=DEV) <= torch.arange(held + beyond - n, held + beyond,
                                                           device=DEV)[:, None]
    if not causal:
        seen = torch.ones_like(seen)
    k, v = (t[c.table[0].long()].flatten(0, 1).double().repeat_interleave(2, 1)
            for t in (c.k, c.v))
    s = torch.einsum("nhe,khe->nhk", q[:n].double(), k) / 8
    p = torch.softmax(s.masked_fill(~seen[:, None], -INF), -1)
    want = torch.einsum("nhk,khe->nhe", p, v)
    size = torch.einsum("nhk,khe->nhe", p, v.abs())
    assert_within(got[:n], want, attention_tolerance(want, size, BF16, held), "beyond")
    want, size = reference(q[n:], c.k, c.v, c.table[1:], kv_lens[1:], q_lens[1:], causal)
    assert_within(got[n:], want, attention_tolerance(want, size, BF16, held), "the other")


@pytest.mark.parametrize("path", PATHS)
def test_pages_outside_the_cache_read_as_zeros(path):
    """Their keys have a score and a value of zero, and their share of the weights."""
    c, q, q_lens, kv_lens = _problem(path)
    c.table[0, 1], c.table[0, 2] = -1, c.pages
    got = _call(c, q, q_lens)
    assert device_status() == FA_ERR_PAGE
    c.k, c.v = (torch.cat([t, torch.zeros_like(t[:1])]) for t in (c.k, c.v))
    c.table[0, 1] = c.pages
    want, size = reference(q, c.k, c.v, c.table, kv_lens, q_lens)
    assert_within(got, want, attention_tolerance(want, size, BF16, max(kv_lens)), path)


@pytest.mark.parametrize("cu,stored", [
    # (sequence, row, place) of lengths 20, 40 and 30
    ([0, 2, 900], [(0, 0, 18), (0, 1, 19), (1, 2, 36), (1, 3, 37), (1, 4, 38), (1, 5, 39)]),
    ([-5, 1, 3], [(0, 0, 19), (1, 1, 38), (1, 2, 39)]),
    ([0, 3, 2 ** 31 - 1], [(0, 0, 17), (0, 1, 18), (0, 2, 19), (1, 3, 37), (1, 4, 38), (1, 5, 39)]),
    # not rising: a row is stored for a sequence that owns it or not at all
    ([4, 1, 3], []),
    ([0, 5, 2, 6], [(0, 0, 15), (0, 1, 16), (2, 5, 29)])])
def test_borders_outside_the_rows_store_what_attention_reads(cu, stored):
    """Borders are held to the packed rows, and tokens stored by what is left of their sequence."""
    lens = [20, 40, 30][:len(cu) - 1]
    c = Cache(lens, 16, 1, 64, BF16, DEV)
    kc, vc = c.k.clone(), c.v.clone()
    k, v = _randn((6, 1, 64), BF16, 4), _randn((6, 1, 64), BF16, 5)
    paged_kv_append(k, v, c.k, c.v, c.table, c.lens,
                    cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV))
    for b, t, place in stored:
        pg, r = _slot(c, b, place)
        kc[pg, r], vc[pg, r] = k[t], v[t]
    assert torch.equal(c.k.nan_to_num(9), kc.nan_to_num(9))
    assert torch.equal(c.v.nan_to_num(9), vc.nan_to_num(9))
    assert device_status() == 0


# --------------------------------------------------------------------------- the status word
def test_a_wait_that_ran_out_outranks_a_bad_page():
    """A bad page leaves a usable result, a wait that gave up does not: the word keeps it."""
    lib = _lib.load()
    c = Cache([20, 40], 16, 1, 64, BF16, DEV, wider=0)
    q, k = _randn((2, 2, 64), BF16), _randn((2, 1, 64), BF16)
    good = c.table.clone()
    c.table[0, 1] = c.pages

    def wait():
        stream = torch.cuda.current_stream(DEV).cuda_stream
        assert lib.fa_selftest_wait_timeout(2000, stream) == 0

    def attend():
        paged_attention(q, c.k, c.v, c.table, c.lens)

    def long():
        c.lens[1] = 60
        attend()
        c.lens[1] = 40

    def append():
        paged_kv_append(k, k, c.k, c.v, c.table, c.lens)

    def chunk():
        _call(Paged(c), q.repeat(20, 4, 1), [20, 20])

    class Paged:
        def __init__(self, c):
            self.k, self.v, self.lens = c.k.repeat(1, 1, 4, 1), c.v.repeat(1, 1, 4, 1), c.lens
            self.table = torch.nn.functional.pad(c.table, (0, 1 << 14), value=-3)

    assert device_status() == 0
    for bad in (attend, long, append, chunk):
        bad()
        assert device_status() == FA_ERR_PAGE and device_status() == 0
        for first, second in ((wait, bad), (bad, wait)):
            first()
            second()
            assert device_status() == FA_ERR_TIMEOUT, bad.__name__
            assert device_status() == 0
    c.table.copy_(good)
