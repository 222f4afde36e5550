"""What the rotary and paged operators refuse, without a GPU: the Python checks on
CPU tensors (devices are checked last) and the C ABI's status codes."""

import struct

import pytest
import torch

from cs348k_fast_attention_grammar_b200 import _lib, paged_attention, paged_kv_append, rotary

BF16 = torch.bfloat16
# The argument structs of include/fa_b200.h: pointers, then 64-bit members.
ROTARY = struct.Struct("=4Q24q")
APPEND = struct.Struct("=11Q35q")
ATTN = struct.Struct("=7Q22qd")
P = 4096            # a stand-in for a device address: argument checks come before any CUDA call


def _z(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def test_rotary_refusals():
    x, pos, f = _z(5, 2, 64), torch.arange(5), torch.ones(32)
    bad = [
        (TypeError, "x must be a torch.Tensor", dict(x=None)),
        (TypeError, "x must be bfloat16 or float16 or float32", dict(x=x.double())),
        (ValueError, "x must be 3-D or 4-D", dict(x=x[0])),
        (ValueError, "contiguous along", dict(x=_z(5, 64, 2).transpose(1, 2))),
        (TypeError, "positions must be int32 or int64", dict(positions=pos.float())),
        (ValueError, "do not match", dict(positions=pos[:4])),
        (ValueError, "do not match", dict(x=_z(3, 2, 5, 64), positions=pos.expand(2, 5))),
        (ValueError, "positions must be 2-D", dict(sections=(16, 16))),
        (ValueError, "do not match", dict(positions=pos.expand(3, 5), sections=(16, 16))),
        (ValueError, "add up to 32", dict(sections=(16, 15))),
        (ValueError, "1 to 4 numbers", dict(sections=(8, 8, 8, 4, 4))),
        (ValueError, "positive whole", dict(sections=(32, 0))),
        (TypeError, "inv_freq must be float32 or float64", dict(inv_freq=f.half())),
        (ValueError, "inv_freq must be 1-D", dict(inv_freq=f[None])),
        (ValueError, "inv_freq must be contiguous", dict(inv_freq=torch.ones(64)[::2])),
        (TypeError, "out must be bfloat16", dict(out=x.float())),
        (ValueError, "x's shape", dict(out=_z(5, 3, 64))),
        (ValueError, "x must be a CUDA tensor", dict()),
    ]
    for kind, text, change in bad:
        with pytest.raises(kind, match=text):
            rotary(**{**dict(x=x, positions=pos, inv_freq=f), **change})


def _append_args(**change):
    return {**dict(k=_z(3, 2, 64), v=_z(3, 2, 64), k_cache=_z(4, 16, 2, 64),
                   v_cache=_z(4, 16, 2, 64), block_table=_z(3, 2, dtype=torch.int32),
                   kv_lens=_ints(1, 2, 3)), **change}


def test_append_refusals():
    f, pos = torch.ones(32), torch.arange(3)
    bad = [
        (TypeError, "k must be bfloat16 or float16", dict(k=_z(3, 2, 64).float())),
        (TypeError, "v must be bfloat16", dict(v=_z(3, 2, 64).half())),
        (ValueError, "shapes differ", dict(v=_z(3, 1, 64))),
        (TypeError, "k_cache must be bfloat16", dict(k_cache=_z(4, 16, 2, 64).half())),
        (ValueError, "caches must both be", dict(k_cache=_z(5, 16, 2, 64))),
        (ValueError, "caches must both be", dict(k_cache=_z(4, 16, 2, 32), v_cache=_z(4, 16, 2, 32))),
        (ValueError, "the caches have 1 heads", dict(k_cache=_z(4, 16, 1, 64),
                                                     v_cache=_z(4, 16, 1, 64))),
        (TypeError, "block_table must be int32", dict(block_table=torch.zeros(3, 2).long())),
        (ValueError, "block_table must be contiguous",
         dict(block_table=_z(2, 3, dtype=torch.int32).T)),
        (ValueError, "kv_lens must be a contiguous", dict(kv_lens=_ints(1, 2))),
        (TypeError, "kv_lens must be int32", dict(kv_lens=pos)),
        (ValueError, "one new token: 3 tokens, 2 sequences",
         dict(block_table=_z(2, 2, dtype=torch.int32), kv_lens=_ints(1, 2))),
        (ValueError, "cu_seqlens must be a contiguous", dict(cu_seqlens=_ints(0, 1, 2))),
        (ValueError, "q must be", dict(q=_z(2, 4, 64))),
        (TypeError, "q must be bfloat16", dict(q=_z(3, 4, 64).half())),
        (ValueError, "q's shape", dict(q=_z(3, 4, 64), q_out=_z(3, 3, 64))),
        (ValueError, "q_out needs q", dict(q_out=_z(3, 4, 64))),
        (ValueError, "need inv_freq", dict(positions=pos)),
        (ValueError, "need inv_freq", dict(sections=(16, 16))),
        (ValueError, "several axes need positions", dict(inv_freq=f, sections=(16, 16))),
        (ValueError, "positions must be", dict(inv_freq=f, positions=pos[:2])),
        (ValueError, "k must be a CUDA tensor", dict()),
    ]
    for kind, text, change in bad:
        with pytest.raises(kind, match=text):
            paged_kv_append(**_append_args(**change))


def test_append_of_no_heads():
    """Queries next to keys of no head have nothing that would write them."""
    none = _z(3, 0, 64)
    with pytest.raises(ValueError, match="at least one head"):
        paged_kv_append(**_append_args(k=none, v=none, k_cache=_z(4, 16, 0, 64),
                                       v_cache=_z(4, 16, 0, 64), q=_z(3, 4, 64)))


def test_attention_refusals():
    good = dict(q=_z(3, 4, 64), k_cache=_z(4, 16, 2, 64), v_cache=_z(4, 16, 2, 64),
                block_table=_z(3, 2, dtype=torch.int32), kv_lens=_ints(1, 2, 3))
    bad = [
        (TypeError, "q must be bfloat16 or float16", dict(q=_z(3, 4, 64).float())),
        (ValueError, "q must be 3-D", dict(q=_z(1, 3, 4, 64))),
        (ValueError, "cannot share", dict(q=_z(3, 3, 64))),
        (ValueError, "cannot share", dict(k_cache=_z(4, 16, 0, 64), v_cache=_z(4, 16, 0, 64))),
        (TypeError, "v_cache must be bfloat16", dict(v_cache=_z(4, 16, 2, 64).half())),
        (ValueError, "max_q_len", dict(max_q_len=-1)),
        (ValueError, "q's shape", dict(out=_z(3, 5, 64))),
        (ValueError, "q must be a CUDA tensor", dict()),
    ]
    for kind, text, change in bad:
        with pytest.raises(kind, match=text):
            paged_attention(**{**good, **change})


def _codes():
    from test_capi import _declared_status_codes
    return _declared_status_codes()


def test_rotary_status_codes():
    lib, code = _lib.load(), _codes()

    def call(x=P, out=P, pos=P, freq=P, dtype=0, B=1, H=2, S=5, D=64, R=64, xs=(640, 320, 64),
             os=(640, 320, 64), axes=1, ends=(32, 0, 0, 0)):
        return lib.fa_rotary(ROTARY.pack(x, out, pos, freq, dtype, B, H, S, D, R, *xs, *os,
                                                axes, *ends, 0, 0, 1, 0, 0, 0, 0), None)

    assert lib.fa_rotary(None, None) == code["FA_ERR_NULL"]
    for name in ("x", "out", "pos", "freq"):
        assert call(**{name: 0}) == code["FA_ERR_NULL"]
    assert call(dtype=3) == call(dtype=-1) == code["FA_ERR_ARG"]
    for change in (dict(B=0), dict(H=-1), dict(S=0), dict(S=1 << 31)):
        assert call(**change) == code["FA_ERR_SHAPE"]
    for change in (dict(D=60), dict(R=24), dict(R=80), dict(R=0), dict(D=2048)):
        assert call(**change) == code["FA_ERR_HEAD_DIM"]
    for change in (dict(axes=0), dict(axes=5), dict(ends=(31, 0, 0, 0)),
                   dict(axes=2, ends=(32, 32, 0, 0))):
        assert call(**change) == code["FA_ERR_ARG"]
    for change in (dict(x=P + 2), dict(out=P + 8), dict(xs=(640, 321, 64)), dict(xs=(640, -64, 64)),
                   dict(os=(640, 0, 64)), dict(dtype=2, xs=(640, 320, 66))):
        assert call(**change) == code["FA_ERR_ALIGN"]


def test_append_status_codes():
    lib, code = _lib.load(), _codes()

    def call(ptrs=(P,) * 11, dtype=0, T=3, B=3, Hq=4, Hkv=2, D=64, R=64, pages=4, page=16, width=2,
             ts=2, st=(128, 64, 128, 64, 256, 64, 256, 64), cs=(2048, 128, 64) * 2, axes=1,
             ends=(32, 0, 0, 0)):
        return lib.fa_paged_append(APPEND.pack(
            *ptrs, dtype, T, B, Hq, Hkv, D, R, pages, page, width, ts, *st, *cs, axes, *ends, 0, 1,
            0, 0, 0), None)

    def without(*which):
        return tuple(0 if i in which else P for i in range(11))

    assert lib.fa_paged_append(None, None) == code["FA_ERR_NULL"]
    for i in (0, 1, 2, 3, 4, 5, 6, 7, 10):
        assert call(ptrs=without(i)) == code["FA_ERR_NULL"]
    assert call(ptrs=without(9), axes=2, ends=(16, 32, 0, 0)) == code["FA_ERR_NULL"]
    assert call(dtype=2) == code["FA_ERR_ARG"]
    for change in (dict(T=0), dict(B=0), dict(Hq=0), dict(Hkv=0), dict(pages=0), dict(width=0),
                   dict(page=8), dict(page=48), dict(page=2048), dict(ptrs=without(8), T=4)):
        assert call(**change) == code["FA_ERR_SHAPE"]
    assert call(ts=1) == code["FA_ERR_STRIDE"]
    for change in (dict(D=60), dict(R=8), dict(R=80)):
        assert call(**change) == code["FA_ERR_HEAD_DIM"]
    assert call(ends=(30, 0, 0, 0)) == code["FA_ERR_ARG"]
    for i in (0, 1, 2, 3, 4, 5):
        ptrs = tuple(P + 2 if j == i else P for j in range(11))
        assert call(ptrs=ptrs) == code["FA_ERR_ALIGN"]
    for i in range(8):
        st = [128, 64, 128, 64, 256, 64, 256, 64]
        st[i] += 4
        assert call(st=st) == code["FA_ERR_ALIGN"]
    assert call(cs=(2048, 0, 64, 2048, 128, 64)) == code["FA_ERR_ALIGN"]


def test_attention_status_codes():
    lib, code = _lib.load(), _codes()

    def call(ptrs=(P,) * 7, dtype=0, T=3, B=3, Hq=4, Hkv=2, D=64, pages=4, page=16, width=2, ts=2,
             st=(256, 64, 256, 64), cs=(2048, 128, 64) * 2, longest=1, scale=0.125):
        args = ATTN.pack(*ptrs, dtype, T, B, Hq, Hkv, D, pages, page, width, ts, *st, *cs,
                                longest, 1, scale)
        rc = lib.fa_paged_attn(args, P, 1 << 40, None)
        assert lib.fa_paged_attn_workspace(args) == -rc
        return rc

    assert lib.fa_paged_attn(None, None, 0, None) == code["FA_ERR_NULL"]
    for i in range(6):
        assert call(ptrs=tuple(0 if j == i else P for j in range(7))) == code["FA_ERR_NULL"]
    for change in (dict(dtype=2), dict(scale=float("inf")), dict(scale=float("nan"))):
        assert call(**change) == code["FA_ERR_ARG"]
    for change in (dict(T=0), dict(B=0), dict(Hq=5), dict(Hkv=0), dict(Hq=258), dict(pages=0),
                   dict(width=0), dict(page=8), dict(page=24), dict(page=2048), dict(longest=0),
                   dict(T=1 << 31), dict(width=1 << 27, ts=1 << 27), dict(ptrs=(P,) * 6 + (0,), T=4)):
        assert call(**change) == code["FA_ERR_SHAPE"]
    for D in (0, 4, 60, 136):
        assert call(D=D) == code["FA_ERR_HEAD_DIM"]
    assert call(ts=1) == code["FA_ERR_STRIDE"]
    for i in range(4):
        assert call(ptrs=tuple(P + 4 if j == i else P for j in range(7))) == code["FA_ERR_ALIGN"]
    for change in (dict(st=(256, 60, 256, 64)), dict(st=(256, 64, 0, 64)),
                   dict(cs=(2048, 130, 64, 2048, 128, 64)), dict(cs=(-2048, 128, 64) * 2)):
        assert call(**change) == code["FA_ERR_ALIGN"]


def test_argument_structs_match_the_header():
    """The packed sizes are those of the C structs (every member is 8 bytes wide)."""
    import os
    import re
    from conftest import ROOT
    text = open(os.path.join(ROOT, "include", "fa_b200.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, packed in (("fa_rotary_args", ROTARY), ("fa_paged_append_args", APPEND),
                         ("fa_paged_attn_args", ATTN)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        n = 0
        for decl in body.split(";"):
            for member in decl.replace("*", "* ").split(","):
                m = re.search(r"(\w+)(?:\[(\d+)\])?\s*$", member.strip())
                if m:
                    n += int(m.group(2) or 1)
        assert packed.size == 8 * n, name


# ---------------------------------------------------------------------------
# The kernels' index arithmetic (csrc/paged.cuh), compiled for the host
# ---------------------------------------------------------------------------
_HARNESS = r"""
#define __host__
#define __device__
#define __forceinline__ inline
#include "paged.cuh"
extern "C" {
int seq_of_row(const int* cu, int B, int t) {
  return fa::seq_of_row(cu, B, t, [&](int lo, int step, int hi) {
    int n = 0;
    for (int lane = 0; lane < 32; ++lane) {
      const int64_t at = lo + static_cast<int64_t>(lane + 1) * step;
      n += at < hi && cu[at] <= t;
    }
    return n;
  });
}
void seq_rows(const int* cu, int b, int T, int* out) {
  const fa::SeqRows r = fa::seq_rows(cu, b, T);
  out[0] = r.begin;
  out[1] = r.end;
}
int page_at(const int* row, int place, int shift, int max_pages, int pages) {
  return fa::page_at(row, place, shift, max_pages, pages);
}
int held_len(int len, int shift, int max_pages) { return fa::held_len(len, shift, max_pages); }
}
"""


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    import ctypes
    import os
    import subprocess
    from conftest import ROOT
    d = tmp_path_factory.mktemp("index")
    src, lib = d / "index.cc", d / "index.so"
    src.write_text(_HARNESS)
    csrc = os.path.join(ROOT, "cs348k_fast_attention_grammar_b200", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-I", csrc, str(src), "-o",
                    str(lib)], check=True)
    return ctypes.CDLL(str(lib))


def _array(values):
    import ctypes
    return (ctypes.c_int * len(values))(*values)


def test_rows_of_sequences(index):
    cu = [2, 5, 5, 5, 9, 10]
    a = _array(cu)
    for t in range(-1, 14):
        want = next((b for b in range(5) if cu[b] <= t < cu[b + 1]), -1)
        assert index.seq_of_row(a, 5, t) == want, t
    for B in (1, 2, 31, 32, 33, 34, 63, 65, 1000, 1056, 1057, 40000):
        cu = [0]
        for b in range(B):
            cu.append(cu[-1] + (b * 7 + B) % 3)
        a = _array(cu)
        owner = {}
        for b in range(B):
            for t in range(cu[b], cu[b + 1]):
                owner[t] = b
        for t in list(range(0, cu[-1], max(1, cu[-1] // 500))) + [cu[-1] - 1, cu[-1], cu[-1] + 1]:
            assert index.seq_of_row(a, B, t) == owner.get(t, -1), (B, t)
    assert [index.seq_of_row(None, 3, t) for t in (0, 2, 3)] == [0, 2, -1]
    out = _array([0, 0])
    for borders, T in (([0, 1, 900], 4), ([-5, 1, 2], 4), ([3, 1, 2], 4), ([0, 2 ** 31 - 1, 1], 4),
                       ([9, 12, -2 ** 31], 4)):
        a = _array(borders)
        for b in range(2):
            index.seq_rows(a, b, T, out)
            assert 0 <= out[0] <= out[1] <= T
            if 0 <= borders[b] <= borders[b + 1] <= T:
                assert list(out) == borders[b:b + 2]
        for t in range(T):
            assert -1 <= index.seq_of_row(a, 2, t) < 2


def test_pages_and_lengths(index):
    row = _array([3, -1, 7, 6, 2 ** 31 - 1, -2 ** 31])
    for place in (-2 ** 31, -1, 0, 15, 16, 31, 32, 47, 48, 64, 80, 95, 96, 2 ** 31 - 1):
        i = place // 16
        want = row[i] if 0 <= i < 6 and 0 <= row[i] < 7 else -1
        assert index.page_at(row, place, 4, 6, 7) == want, place
    for n in (-2 ** 31, -1, 0, 1, 95, 96, 97, 2 ** 31 - 1):
        assert index.held_len(n, 4, 6) == min(max(n, 0), 96)
    # a table of more places than an int counts
    assert index.held_len(2 ** 31 - 1, 10, 2 ** 31 - 1) == 2 ** 31 - 1
