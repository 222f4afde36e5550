// Rotary positions, alone (fa_rotary) and on the way into a paged key/value
// cache (fa_paged_append):
//     (a, b) -> (a cos t - b sin t, b cos t + a sin t),   t = position * inv_freq[i]
//
// Both are bound by HBM: each value is read once and written once.  A CTA of
// 192 threads takes a few rows (tokens).  It loads its first vectors, finds the
// rows' places and computes their sines and cosines once into shared memory while
// those loads are in flight, then rotates and stores; a thread's item is two
// 16-byte vectors R / 2 channels apart, so that the planes (i, i + R / 2) stay
// inside one thread and the planes (2i, 2i + 1) inside one vector.  Every head of
// a row shares the row's angles.
//
// Measured: 16384 tokens of 32 heads of 128 bf16 channels turned by three axes in
// 42.8 us, 6.28 TB/s (45.2 when nothing else runs for a second, with a lower clock);
// 4636 tokens of 16 heads, 64 of 128 channels turned, appended
// with their queries in 21.5 to 22.8 us, 5.1 TB/s (one wave of CTAs, which starts with its
// rows' places: a search in the borders, a length, a table entry); one token, 4 us,
// the launch.
//
// An angle of a far position needs more than fp32: position * inv_freq is
// formed in fp64 in turns (inv_freq / 2 pi), the whole turns are dropped
// exactly, and the remainder (at most half a turn) goes to sincospif in fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fa_internal.h"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace fa {
namespace {

constexpr int kRotThreads = 192;        // 192 x 4 items: 3 rows of 256 items, 6 of 128
// Items of a thread whose loads are in flight together, and CTAs per SM (by
// registers).  16384 tokens of 32 heads of 128 channels turned: 44.5 us with 1 item
// and 8 CTAs, 43.6 with 2 and 6, 45.9 with 2 and 5; 4636 tokens of 16 heads appended
// with their queries, whose CTAs first wait for their rows' places: 23.1, 25.0, 29.0.
constexpr int rot_ahead(bool append) { return append ? 1 : 2; }
constexpr int rot_ctas_per_sm(bool append) { return append ? 8 : 6; }
// Goes of a CTA over its items: a row's place takes a chain of loads that the goes
// of an append share (those tokens: 24.8 us with 2, 23.0 with 4, 22.4 with 8; the
// rotation alone 57.7, 43.6, 46.8).
constexpr int rot_batches(bool append) { return append ? 8 : 4; }
constexpr int kRotMaxRows = 64;         // rows of one CTA
constexpr int kRotMaxAngles = 2048;     // angles of one CTA (16 KiB of shared memory)

struct Angles {
  const void* pos;
  const void* freq;
  int64_t pos_sa, pos_sb, pos_ss;       // elements: axis, batch, row
  int sec_end[4];
  int axes, R, pos64, freq64;
  float sign;                           // -1 turns the other way
};

// One tensor's head vectors of a row: `heads` of them, rotated or copied.
struct Part {
  const void* src;
  void* dst;
  int64_t src_sb, src_sh, src_ss;       // elements
  int64_t dst_sb, dst_sh, dst_ss;
  int heads, rotate;
  int items, count;                     // items of a head, of all heads
  unsigned by_items;                    // reciprocal of items, for quotient()
};

struct RotParams {
  Angles ang;
  Part part[3];                         // append: keys, values, queries; rotary: one part
  int parts, D;
  int64_t rows;
  int S;                                // rows of one batch entry
  int rows_per_cta, items_per_row;
  unsigned by_row;                      // reciprocal of items_per_row
  // append only
  const int32_t* table;
  const int32_t* kv_lens;
  const int32_t* cu;
  int B, pages, page_shift, max_pages;
  int64_t table_stride;
  int64_t kc_page, vc_page;             // cache page strides (elements)
  int* status;
};

template <int TYPE>
struct Elem;                            // TYPE: fa_dtype
template <>
struct Elem<FA_BF16> {
  static constexpr int kSize = 2;
};
template <>
struct Elem<FA_F16> {
  static constexpr int kSize = 2;
};
template <>
struct Elem<FA_F32> {
  static constexpr int kSize = 4;
};

template <int TYPE>
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[16 / Elem<TYPE>::kSize]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (TYPE == FA_F32) {
      f[i] = __uint_as_float(w[i]);
    } else {
      f[2 * i] = unpack_16<TYPE == FA_F16>(w[i], false);
      f[2 * i + 1] = unpack_16<TYPE == FA_F16>(w[i], true);
    }
  }
}

template <int TYPE>
__device__ __forceinline__ uint4 pack(const float (&f)[16 / Elem<TYPE>::kSize]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (TYPE == FA_F32) w[i] = __float_as_uint(f[i]);
    else w[i] = pack_16x2<TYPE == FA_F16>(f[2 * i], f[2 * i + 1]);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// N consecutive cosines or sines from shared memory.
template <int N>
__device__ __forceinline__ void load_angles(const float* at, float (&f)[N]) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(at + i);
      f[i] = v.x;
      f[i + 1] = v.y;
      f[i + 2] = v.z;
      f[i + 3] = v.w;
    }
  } else {
    const float2 v = *reinterpret_cast<const float2*>(at);
    f[0] = v.x;
    f[1] = v.y;
  }
}

__device__ __forceinline__ float2 cos_sin(const Angles& a, int64_t b, int64_t s, int i,
                                          bool own_pos, int place) {
  double pos;
  if (own_pos) {
    pos = static_cast<double>(place);
  } else {
    int axis = 0;
    while (axis + 1 < a.axes && i >= a.sec_end[axis]) ++axis;
    const int64_t at = axis * a.pos_sa + b * a.pos_sb + s * a.pos_ss;
    pos = a.pos64 ? static_cast<double>(static_cast<const int64_t*>(a.pos)[at])
                  : static_cast<double>(static_cast<const int32_t*>(a.pos)[at]);
  }
  const double f = a.freq64 ? static_cast<const double*>(a.freq)[i]
                            : static_cast<double>(static_cast<const float*>(a.freq)[i]);
  const double turns = pos * (f * 0.15915494309189535);
  float2 cs;
  sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &cs.y, &cs.x);
  cs.y *= a.sign;
  return cs;
}

// n / d by the reciprocal r = floor(2^32 / d) + 1, exact while n d < 2^32; r = 0
// divides (see reciprocal()).
__device__ __forceinline__ unsigned quotient(unsigned n, unsigned d, unsigned r) {
  return r != 0 ? __umulhi(n, r) : n / d;
}

// An item: up to two vectors of one head.
struct Item {
  const char* src;
  char* dst;            // its tensor's start; the row's offset is added when it is known
  int off0, off1;       // byte offsets of the vectors, -1: no second one
  int row, angle;       // row of the CTA; first plane, -1: copied
  int part;
};

// APPEND: rows are packed new tokens, keys and values go to their pages.
template <int TYPE, bool APPEND, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotThreads, rot_ctas_per_sm(APPEND))
    rotary_kernel(const RotParams p) {
  constexpr int kSize = Elem<TYPE>::kSize;
  constexpr int V = 16 / kSize;
  __shared__ __align__(16) float s_cos[kRotMaxAngles], s_sin[kRotMaxAngles];
  __shared__ int64_t s_dst[3][kRotMaxRows];     // element offset of the row's place, -1: none
  __shared__ int64_t s_batch[kRotMaxRows];
  __shared__ int s_place[kRotMaxRows];
  grid_dependency_wait();

  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * p.rows_per_cta;
  const int rows = static_cast<int>(min(static_cast<int64_t>(p.rows_per_cta), p.rows - row0));
  const int half = p.ang.R / 2;
  const unsigned rot_items = half / V;
  const unsigned total = rows * p.items_per_row;

  if (!APPEND) {
    if (threadIdx.x < rows) s_batch[threadIdx.x] = (row0 + threadIdx.x) / p.S;
    __syncthreads();
  }

  auto locate = [&](unsigned it) {
    Item x;
    x.row = quotient(it, p.items_per_row, p.by_row);
    unsigned r = it - x.row * p.items_per_row;
    x.part = 0;
    if (APPEND) {
      while (x.part + 1 < p.parts && r >= static_cast<unsigned>(p.part[x.part].count)) {
        r -= p.part[x.part].count;
        ++x.part;
      }
    }
    const Part& q = p.part[x.part];
    const unsigned head = quotient(r, q.items, q.by_items);
    const unsigned chunk = r - head * q.items;
    const int64_t b = APPEND ? 0 : s_batch[x.row];
    const int64_t s = row0 + x.row - b * p.S;
    x.src = static_cast<const char*>(q.src) +
            (b * q.src_sb + s * q.src_ss + head * q.src_sh) * kSize;
    x.dst = static_cast<char*>(q.dst) + head * q.dst_sh * kSize;
    if (!APPEND) x.dst += (b * q.dst_sb + s * q.dst_ss) * kSize;
    if (q.rotate && chunk < rot_items) {
      x.off0 = chunk * 16;
      x.off1 = (half + chunk * V) * kSize;
      x.angle = x.row * half + chunk * (INTERLEAVED ? V / 2 : V);
    } else {
      const int c0 = q.rotate ? p.ang.R + (chunk - rot_items) * V : chunk * V;
      const int c1 = c0 + (q.items - (q.rotate ? rot_items : 0)) * V;
      x.off0 = c0 * kSize;
      x.off1 = c1 < p.D ? c1 * kSize : -1;
      x.angle = -1;
    }
    return x;
  };
  auto load = [&](const Item& x, uint4& u0, uint4& u1) {
    u0 = *reinterpret_cast<const uint4*>(x.src + x.off0);
    if (x.off1 >= 0) u1 = *reinterpret_cast<const uint4*>(x.src + x.off1);
  };

  // The first items' loads are in flight while places and angles are found.
  constexpr bool kTwo = rot_ahead(APPEND) == 2;
  unsigned it = threadIdx.x;
  uint4 a, c, a1, c1;
  Item item, item1;
  if (it < total) {
    item = locate(it);
    load(item, a, c);
  }
  if (kTwo && it + kRotThreads < total) {
    item1 = locate(it + kRotThreads);
    load(item1, a1, c1);
  }
  if (APPEND) {
    // Where each row goes: one warp per row.
    const int lane = threadIdx.x & 31;
    for (int r = threadIdx.x >> 5; r < rows; r += kRotThreads / 32) {
      const int t = static_cast<int>(row0) + r;
      const int b = seq_of_row(p.cu, p.B, t, [&](int lo, int step, int hi) {
        const int64_t at = lo + static_cast<int64_t>(lane + 1) * step;
        return __popc(__ballot_sync(0xffffffffu, at < hi && p.cu[at < hi ? at : lo] <= t));
      });
      if (lane == 0) {
        // (borders that are not rising may lead to a sequence without this row)
        const int len = b < 0 ? 0 : p.kv_lens[b];
        const SeqRows sr = b < 0 ? SeqRows{0, 0} : seq_rows(p.cu, b, static_cast<int>(p.rows));
        const bool owned = sr.begin <= t && t < sr.end;
        int64_t k = -1, v = -1;
        int place = 0;
        if (owned) {
          place = max(len, 0) - (sr.end - t);
          if (place >= 0) {
            const int page = page_at(p.table + b * p.table_stride, place, p.page_shift,
                                     p.max_pages, p.pages);
            if (page >= 0) {
              const int in = place & ((1 << p.page_shift) - 1);
              k = page * p.kc_page + in * p.part[0].dst_ss;
              v = page * p.vc_page + in * p.part[1].dst_ss;
            } else {
              atomicMax(p.status, kDevBadPage);
            }
          }
        }
        s_dst[0][r] = k;
        s_dst[1][r] = v;
        s_dst[2][r] = owned ? t * p.part[2].dst_ss : -1;
        s_place[r] = place;
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < rows * half; i += kRotThreads) {
    const int r = static_cast<unsigned>(i) / static_cast<unsigned>(half);
    const int64_t b = APPEND ? 0 : s_batch[r];
    if (APPEND && s_dst[2][r] < 0) continue;           // (a row of no sequence has no position)
    const float2 w = cos_sin(p.ang, b, row0 + r - b * p.S, i - r * half, p.ang.pos == nullptr,
                             APPEND ? s_place[r] : 0);
    s_cos[i] = w.x;
    s_sin[i] = w.y;
  }
  __syncthreads();

  auto finish = [&](const Item& x, const uint4& u0, const uint4& u1) {
    char* dst = x.dst;
    if (APPEND) {
      const int64_t at = s_dst[x.part][x.row];
      if (at < 0) return;
      dst += at * kSize;
    }
    if (x.angle < 0) {
      *reinterpret_cast<uint4*>(dst + x.off0) = u0;
      if (x.off1 >= 0) *reinterpret_cast<uint4*>(dst + x.off1) = u1;
      return;
    }
    float f[V], g[V];
    unpack<TYPE>(u0, f);
    unpack<TYPE>(u1, g);
    if (INTERLEAVED) {
      float cf[V / 2], sf[V / 2], cg[V / 2], sg[V / 2];
      load_angles(s_cos + x.angle, cf);
      load_angles(s_sin + x.angle, sf);
      load_angles(s_cos + x.angle + half / 2, cg);
      load_angles(s_sin + x.angle + half / 2, sg);
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float f0 = f[e], g0 = g[e];
        f[e] = fmaf(f0, cf[e / 2], -f[e + 1] * sf[e / 2]);
        f[e + 1] = fmaf(f[e + 1], cf[e / 2], f0 * sf[e / 2]);
        g[e] = fmaf(g0, cg[e / 2], -g[e + 1] * sg[e / 2]);
        g[e + 1] = fmaf(g[e + 1], cg[e / 2], g0 * sg[e / 2]);
      }
    } else {
      float co[V], si[V];
      load_angles(s_cos + x.angle, co);
      load_angles(s_sin + x.angle, si);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float f0 = f[e];
        f[e] = fmaf(f0, co[e], -g[e] * si[e]);
        g[e] = fmaf(g[e], co[e], f0 * si[e]);
      }
    }
    *reinterpret_cast<uint4*>(dst + x.off0) = pack<TYPE>(f);
    *reinterpret_cast<uint4*>(dst + x.off1) = pack<TYPE>(g);
  };
  while (it < total) {
    finish(item, a, c);
    if (kTwo && it + kRotThreads < total) finish(item1, a1, c1);
    it += rot_ahead(APPEND) * kRotThreads;
    if (it < total) {
      item = locate(it);
      load(item, a, c);
    }
    if (kTwo && it + kRotThreads < total) {
      item1 = locate(it + kRotThreads);
      load(item1, a1, c1);
    }
  }
}

// For quotients of numbers up to most: 0 where they would not be exact (d = 1
// among them, whose reciprocal takes 33 bits).
unsigned reciprocal(int64_t d, int64_t most) {
  return d > 1 && most * d < (int64_t{1} << 32) ? static_cast<unsigned>(0xffffffffu / d + 1) : 0;
}

int launch_rotary(RotParams& p, int dtype, bool append, bool interleaved, cudaStream_t stream) {
  int dev = 0;
  const int rc = prepare_device(nullptr, 0, &dev);
  if (rc != FA_OK) return rc;
  const int V = dtype == FA_F32 ? 4 : 8;
  const int half = p.ang.R / 2;
  p.items_per_row = 0;
  for (int i = 0; i < p.parts; ++i) {
    Part& q = p.part[i];
    const int rest = q.rotate ? p.D - p.ang.R : p.D;
    q.items = (q.rotate ? half / V : 0) + (rest / V + 1) / 2;
    q.count = q.heads * q.items;
    p.items_per_row += q.count;
  }
  // Rows per CTA: at most what its threads take in rot_batches() goes, within the
  // shared memory for their angles, and so many that the CTAs fill whole waves of
  // the device (the appended tokens above: 26.3 us in 1.3 waves, 23.7 in two).
  int rows = rot_batches(append) * kRotThreads / p.items_per_row;
  if (half > 0) rows = rows < kRotMaxAngles / half ? rows : kRotMaxAngles / half;
  rows = rows < kRotMaxRows ? rows : kRotMaxRows;
  if (rows < 1) rows = 1;
  const int64_t wave =
      static_cast<int64_t>(rot_ctas_per_sm(append)) * (sm_count(dev) > 0 ? sm_count(dev) : 1);
  const int64_t waves = (p.rows + rows * wave - 1) / (rows * wave);
  p.rows_per_cta = static_cast<int>((p.rows + waves * wave - 1) / (waves * wave));
  p.by_row = reciprocal(p.items_per_row, static_cast<int64_t>(p.rows_per_cta) * p.items_per_row);
  for (int i = 0; i < p.parts; ++i)
    p.part[i].by_items = reciprocal(p.part[i].items, p.items_per_row);
  const int64_t grid = (p.rows + p.rows_per_cta - 1) / p.rows_per_cta;
  if (grid > 0x7fffffffLL) return FA_ERR_SHAPE;
  const unsigned g = static_cast<unsigned>(grid);
  if (append) {
    p.status = device_status_ptr();
    if (p.status == nullptr) return FA_ERR_CUDA;
  }
  // (as a programmatic dependent: its CTAs come up as the kernel before ends)
#define FA_ROT(T, A, I) launch_after(rotary_kernel<T, A, I>, dim3(g), kRotThreads, 0, 1, stream, p)
  if (append) {
    if (dtype == FA_BF16)
      return interleaved ? FA_ROT(FA_BF16, true, true) : FA_ROT(FA_BF16, true, false);
    return interleaved ? FA_ROT(FA_F16, true, true) : FA_ROT(FA_F16, true, false);
  }
  if (dtype == FA_BF16)
    return interleaved ? FA_ROT(FA_BF16, false, true) : FA_ROT(FA_BF16, false, false);
  if (dtype == FA_F16)
    return interleaved ? FA_ROT(FA_F16, false, true) : FA_ROT(FA_F16, false, false);
  return interleaved ? FA_ROT(FA_F32, false, true) : FA_ROT(FA_F32, false, false);
#undef FA_ROT
}

constexpr int64_t kMaxDim = 0x7fffffffLL;

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Strides of `n` dimensions of the given sizes: multiples of 16 bytes where the
// dimension has more than one entry, not negative, and not 0 where written.
bool strides_ok(const int64_t* st, const int64_t* sizes, int n, int elem, bool written) {
  for (int i = 0; i < n; ++i)
    if (sizes[i] > 1 && (st[i] < (written ? 1 : 0) || (st[i] * elem) % 16 != 0)) return false;
  return true;
}

int check_sections(int64_t axes, const int64_t* end, int64_t R) {
  if (axes < 1 || axes > 4) return FA_ERR_ARG;
  int64_t last = 0;
  for (int a = 0; a < axes; ++a) {
    if (end[a] <= last) return FA_ERR_ARG;
    last = end[a];
  }
  return last == R / 2 ? FA_OK : FA_ERR_ARG;
}

void set_angles(Angles& a, const void* pos, const void* freq, int64_t axes, const int64_t* end,
                int64_t R, int64_t pos64, int64_t freq64, bool inverse) {
  a.pos = pos;
  a.freq = freq;
  a.axes = static_cast<int>(axes);
  for (int i = 0; i < 4; ++i) a.sec_end[i] = i < axes ? static_cast<int>(end[i]) : 0;
  a.R = static_cast<int>(R);
  a.pos64 = pos64 != 0;
  a.freq64 = freq64 != 0;
  a.sign = inverse ? -1.f : 1.f;
}

}  // namespace
}  // namespace fa

extern "C" int fa_rotary(const fa_rotary_args* a, void* stream) {
  using namespace fa;
  if (!a || !a->x || !a->out || !a->positions || !a->inv_freq) return FA_ERR_NULL;
  if (a->dtype < FA_BF16 || a->dtype > FA_F32) return FA_ERR_ARG;
  if (a->B <= 0 || a->H <= 0 || a->S <= 0 || a->B > kMaxDim || a->H > 65536 || a->S > kMaxDim)
    return FA_ERR_SHAPE;
  if (a->D < 16 || a->D > 1024 || a->D % 8 || a->R < 16 || a->R > a->D || a->R % 16)
    return FA_ERR_HEAD_DIM;
  const int rc = check_sections(a->axes, a->section_end, a->R);
  if (rc != FA_OK) return rc;
  const int elem = a->dtype == FA_F32 ? 4 : 2;
  const int64_t sizes[3] = {a->B, a->H, a->S};
  if (!strides_ok(a->x_strides, sizes, 3, elem, false) ||
      !strides_ok(a->out_strides, sizes, 3, elem, true) ||
      !aligned16(a->x) || !aligned16(a->out))
    return FA_ERR_ALIGN;
  RotParams p = {};
  set_angles(p.ang, a->positions, a->inv_freq, a->axes, a->section_end, a->R, a->pos_is_i64,
             a->freq_is_f64, a->inverse != 0);
  p.ang.pos_sa = a->pos_strides[0];
  p.ang.pos_sb = a->pos_strides[1];
  p.ang.pos_ss = a->pos_strides[2];
  p.parts = 1;
  p.part[0] = {a->x, a->out, a->x_strides[0], a->x_strides[1], a->x_strides[2],
               a->out_strides[0], a->out_strides[1], a->out_strides[2],
               static_cast<int>(a->H), 1, 0, 0};
  p.D = static_cast<int>(a->D);
  p.rows = a->B * a->S;
  p.S = static_cast<int>(a->S);
  return launch_rotary(p, static_cast<int>(a->dtype), false, a->interleaved != 0,
                       static_cast<cudaStream_t>(stream));
}

extern "C" int fa_paged_append(const fa_paged_append_args* a, void* stream) {
  using namespace fa;
  if (!a || !a->k || !a->v || !a->k_cache || !a->v_cache || !a->block_table || !a->kv_lens)
    return FA_ERR_NULL;
  if ((a->R > 0 && !a->inv_freq) || (a->q != nullptr) != (a->q_out != nullptr)) return FA_ERR_NULL;
  if (a->dtype != FA_BF16 && a->dtype != FA_F16) return FA_ERR_ARG;
  if (a->T <= 0 || a->B <= 0 || a->Hkv <= 0 || a->T > kMaxDim || a->B >= kMaxDim ||
      a->Hkv > 65536 || (a->q && (a->Hq <= 0 || a->Hq > 65536)))
    return FA_ERR_SHAPE;
  if (!a->cu_seqlens && a->T != a->B) return FA_ERR_SHAPE;
  if (a->D < 8 || a->D > 1024 || a->D % 8 || a->R < 0 || a->R > a->D || a->R % 16)
    return FA_ERR_HEAD_DIM;
  if (a->pages <= 0 || a->pages > kMaxDim || a->max_pages <= 0 || a->max_pages > kMaxDim ||
      a->page_size < 16 || a->page_size > 1024 || (a->page_size & (a->page_size - 1)))
    return FA_ERR_SHAPE;
  if (a->B > 1 && a->table_stride < a->max_pages) return FA_ERR_STRIDE;
  if (a->R > 0) {
    const int rc = check_sections(a->axes, a->section_end, a->R);
    if (rc != FA_OK) return rc;
    if (a->axes > 1 && !a->positions) return FA_ERR_NULL;
  }
  const int64_t ks[2] = {a->T, a->Hkv}, qs[2] = {a->T, a->Hq};
  const int64_t cs[3] = {a->pages, a->page_size, a->Hkv};
  if (!strides_ok(a->k_strides, ks, 2, 2, false) || !strides_ok(a->v_strides, ks, 2, 2, false) ||
      !strides_ok(a->k_cache_strides, cs, 3, 2, true) ||
      !strides_ok(a->v_cache_strides, cs, 3, 2, true) ||
      !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->k_cache) || !aligned16(a->v_cache))
    return FA_ERR_ALIGN;
  if (a->q && (!strides_ok(a->q_strides, qs, 2, 2, false) ||
               !strides_ok(a->q_out_strides, qs, 2, 2, true) || !aligned16(a->q) || !aligned16(a->q_out)))
    return FA_ERR_ALIGN;
  RotParams p = {};
  set_angles(p.ang, a->positions, a->inv_freq, a->axes, a->section_end, a->R, a->pos_is_i64,
             a->freq_is_f64, false);
  p.ang.pos_sa = a->pos_strides[0];
  p.ang.pos_ss = a->pos_strides[1];
  const int rotate = a->R > 0;
  p.part[0] = {a->k, a->k_cache, 0, a->k_strides[1], a->k_strides[0], 0, a->k_cache_strides[2],
               a->k_cache_strides[1], static_cast<int>(a->Hkv), rotate, 0, 0};
  p.part[1] = {a->v, a->v_cache, 0, a->v_strides[1], a->v_strides[0], 0, a->v_cache_strides[2],
               a->v_cache_strides[1], static_cast<int>(a->Hkv), 0, 0, 0};
  p.parts = 2;
  if (a->q) {
    p.part[2] = {a->q, a->q_out, 0, a->q_strides[1], a->q_strides[0], 0, a->q_out_strides[1],
                 a->q_out_strides[0], static_cast<int>(a->Hq), rotate, 0, 0};
    p.parts = 3;
  }
  p.D = static_cast<int>(a->D);
  p.rows = a->T;
  p.S = static_cast<int>(a->T);
  p.table = a->block_table;
  p.kv_lens = a->kv_lens;
  p.cu = a->cu_seqlens;
  p.B = static_cast<int>(a->B);
  p.pages = static_cast<int>(a->pages);
  p.page_shift = __builtin_ctzll(static_cast<unsigned long long>(a->page_size));
  p.max_pages = static_cast<int>(a->max_pages);
  p.table_stride = a->table_stride;
  p.kc_page = a->k_cache_strides[0];
  p.vc_page = a->v_cache_strides[0];
  return launch_rotary(p, static_cast<int>(a->dtype), true, a->interleaved != 0,
                       static_cast<cudaStream_t>(stream));
}
