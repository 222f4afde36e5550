// Attention of new tokens over a paged key/value cache (fa_paged_attn):
//     o = softmax(q K^T * scale) V      per token and head
//
// Query heads that share a key/value head are rows of one tile together with
// the sequence's new tokens: row r of a sequence is token r / g, head r % g of
// the group (g = Hq / Hkv), so each key is read once for all of them.
//
// paged_rows_kernel takes sequences of few rows (a generation step).  It is
// bound by HBM: two passes' worth of arithmetic per key and row is far below
// what even warp-level matrix instructions deliver (tcgen05 would put its 16 rows
// into tiles of 128), so the kernel is built around its loads.  A CTA has four warps
// (more for short tables, below); per 64-key block each warp owns 16 keys, loads
// their K and V rows with 16-byte asynchronous copies into a ring of its own (no
// barrier between warps), and keeps its own running maximum, sum and output, joined
// over the warps when the CTA leaves a tile.  32 sequences of up to 8192 keys, 32/8
// heads of 128: 109 to 111 us, 6.2 TB/s; 3 of up to 131072, 32/4 heads: 103 to 106
// us, 6.1 TB/s.  The weights are rounded to the 16-bit type that the matrix
// instructions take; their sum is of the unrounded ones, in fp32 like the output.
//
// CTAs work in teams of up to 16 key heads, a head each, that walk the same keys
// side by side: a cached token's heads lie next to each other, and DRAM is read
// in longer runs than one head's row (64 sequences of up to 4096 keys, 8 heads of
// 64: 4127 -> 5344 GB/s; D = 128: 6071 -> 6136).  The key blocks
// of all (sequence, group of heads, row tile) units, one after the other, are cut
// into equal ranges, one per team, whatever the lengths: a unit that crosses a
// range's border leaves (m, l, O) of its parts in the workspace and
// paged_rows_join adds them up in an order of their own, so results do not depend
// on timing.
//
// Neither kernel lets its dependents start before it ends: CTAs that wait beside it
// cost more than they save (32 sequences of up to 8192 keys, 16 heads of 64: 138
// us with early starts, where the next call's CTAs then all begin at one moment, 112
// without; 3 of up to 131072, 32/4 heads of 128: 106.2, 104.7).
#include <cuda_bf16.h>

#include <atomic>
#include <cmath>

#include "paged_attn.h"
#include "sm100_2sm.cuh"

namespace fa {
namespace {

// ---------------------------------------------------------------------------
// Schedule of the row kernel
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 128;
constexpr int kRowWarps = 4;
constexpr int kRowKeys = 64;            // keys of a block: 16 per warp

// A sequence's row tiles and key blocks.
struct RowWork : SeqWork {
  int tiles, blocks;
};

__device__ __forceinline__ RowWork row_work(const PagedParams& p, int b, int tile_rows) {
  RowWork w;
  static_cast<SeqWork&>(w) = seq_work(p, b);
  w.tiles = static_cast<int>((static_cast<int64_t>(w.q_len) * p.g + tile_rows - 1) / tile_rows);
  w.blocks = max(1, (w.kv_len + kRowKeys - 1) / kRowKeys);
  return w;
}
__device__ __forceinline__ int64_t weight(const PagedParams& p, const RowWork& w) {
  return static_cast<int64_t>(w.tiles) * (p.Hkv / p.team) * w.blocks;
}

// The sum of v over the CTA's threads below this one, and over all of them.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* red, int64_t* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) red[w] = x;
  __syncthreads();
  int64_t before = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < kRowWarps; ++i) {
    if (i < w) before += red[i];
    sum += red[i];
  }
  *total = sum;
  return before + x - v;
}

// A team's range [start, end) of the key blocks and the sequence that it starts in.
struct Range {
  int64_t start, end, per;
  int64_t base;          // first key block of sequence b
  int b;
  RowWork work;          // of sequence b
};

__device__ __forceinline__ Range find_range(const PagedParams& p, int team, int tile_rows) {
  __shared__ int64_t red[kRowWarps];
  __shared__ int64_t s_base;
  __shared__ int s_b;
  __shared__ RowWork s_work;
  Range r;
  int64_t total = 0;
  RowWork first = {};                         // the first kRowThreads sequences': kept
  int64_t first_before = 0;
  for (int b0 = 0; b0 < p.B; b0 += kRowThreads) {
    const int b = b0 + threadIdx.x;
    RowWork w = {};
    if (b < p.B) w = row_work(p, b, tile_rows);
    int64_t sum;
    const int64_t before = block_scan(weight(p, w), red, &sum);
    if (b0 == 0) {
      first = w;
      first_before = before;
    }
    total += sum;
  }
  r.per = max(static_cast<int64_t>(p.min_blocks), (total + p.ctas - 1) / p.ctas);
  r.start = min(total, r.per * team);
  r.end = min(total, r.start + r.per);
  if (threadIdx.x == 0) s_b = p.B;
  __syncthreads();
  if (r.start < r.end) {
    int64_t base = 0;
    for (int b0 = 0; b0 < p.B; b0 += kRowThreads) {
      const int b = b0 + threadIdx.x;
      RowWork w = first;
      int64_t before = first_before, sum = 0;
      if (p.B > kRowThreads) {
        w = {};
        if (b < p.B) w = row_work(p, b, tile_rows);
        before = block_scan(weight(p, w), red, &sum);
      }
      if (base + before <= r.start && r.start < base + before + weight(p, w)) {
        s_b = b;
        s_base = base + before;
        s_work = w;
      }
      base += sum;
    }
  }
  __syncthreads();
  r.b = s_b;
  r.base = s_base;
  r.work = s_work;
  return r;
}

// ---------------------------------------------------------------------------
// Warp-level pieces
// ---------------------------------------------------------------------------
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  if (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A value from the shared memory of CTA `cta` of the cluster, at this CTA's address.
__device__ __forceinline__ float cluster_load(uint32_t addr, int cta) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(cta));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t addr, int cta) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(cta));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

// How a launch cuts its work: ranges of key blocks for teams of CTAs, joined
// afterwards; a CTA per sequence, head and row tile; the same with more warps,
// and a cluster of up to 8 CTAs instead of one, for fewer CTAs than SMs, where a
// warp's chain of 16-key steps (about 900 clocks each with one warp per scheduler)
// is what a call waits for.  The cluster's CTAs take turns at the steps and add
// their results up through each other's shared memory.
enum Cut { kSplit, kWhole, kWholeWide };

template <int DT, int MT, Cut CUT = kSplit>
struct RowCfg {
  static constexpr int kRows = 16 * MT;
  static constexpr int kWarps = CUT == kWholeWide ? (DT == 64 ? 16 : 8) : kRowWarps;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kStep = 16 * kWarps;              // keys of the CTA's steps
  static constexpr int kStepLog2 = kWarps == 16 ? 8 : kWarps == 8 ? 7 : 6;
  static_assert(1 << kStepLog2 == kStep, "steps are powers of two");
  // Ring steps by shared memory (CTAs per SM also by registers).
  static constexpr int kStages = DT == 64 && MT == 2 ? 6 : 3;
  static constexpr int kCtasPerSm = CUT == kWholeWide ? 1 : DT == 64 && MT == 1 ? 4 : 2;
  static constexpr int kTile = 16 * DT * 2;              // 16 keys of K or of V
  static constexpr int kStage = 2 * kTile;
  static constexpr int kWarp = kStages * kStage;
  static constexpr int kRing = kWarps * kWarp;
  static constexpr int kSlot = kRows * (DT + 2);         // floats of a partial result
  static constexpr int kSumOff = kRing + 2 * kWarps * kRows * 4;   // m, l of each warp before it
  static constexpr int kSmem = kSumOff + (CUT == kWholeWide ? kSlot * 4 : 0);
  static_assert(kWarps * kRows * DT * 4 <= kRing, "the joined output reuses the ring");
};

template <int DT, int MT, bool F16, Cut CUT>
__global__ void __launch_bounds__(RowCfg<DT, MT, CUT>::kThreads, RowCfg<DT, MT, CUT>::kCtasPerSm)
    paged_rows_kernel(const PagedParams p) {
  using C = RowCfg<DT, MT, CUT>;
  constexpr bool WHOLE = CUT != kSplit;   // teams of all heads, a sequence each
  constexpr int CH = DT / 8;            // 16-byte chunks of a row
  constexpr int RPI = 32 / CH;          // rows one warp-wide copy covers
  extern __shared__ __align__(128) uint8_t smem[];
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = smem_u32(smem) + warp * C::kWarp;
  float* s_o = reinterpret_cast<float*>(smem);
  float* s_m = reinterpret_cast<float*>(smem + C::kRing);
  float* s_l = s_m + C::kWarps * C::kRows;

  Range rg = {};
  int tile = 0;                         // whole units: this CTA's row tile
  int ahead = 0;                        // and a page, loaded along with the lengths
  // This warp's first key of a block or unit, and how far its steps are apart.
  const int cshift = CUT == kWholeWide ? p.cluster_shift : 0;
  const int cluster = 1 << cshift;
  const unsigned rank = blockIdx.x & (cluster - 1), cta = blockIdx.x >> cshift;
  const int warp_key = (rank * C::kWarps + warp) * 16;
  const int step_keys = C::kStep << cshift;
  if (WHOLE) {
    const unsigned team = cta / static_cast<unsigned>(p.team);
    rg.b = team / static_cast<unsigned>(p.tile_ctas);
    tile = team - rg.b * p.tile_ctas;
    const int at = (warp_key + lane * step_keys) >> p.page_shift;
    if (at < p.max_pages) ahead = p.table[rg.b * p.table_stride + at];
    rg.work = row_work(p, rg.b, C::kRows);
  } else {
    rg = find_range(p, cta / p.team, C::kRows);
    if (rg.start >= rg.end) {
      if (threadIdx.x == 0) p.open[cta].parts = 0;
      return;
    }
  }
  const int page_mask = (1 << p.page_shift) - 1;
  const int crow = lane / CH, cchunk = lane % CH;
  const bool cin = cchunk * 8 < p.D;
  const char* const kc = static_cast<const char*>(p.kc);
  const char* const vc = static_cast<const char*>(p.vc);

  int b = rg.b;
  int64_t base = rg.base, cur = rg.start;
  RowWork w = rg.work;
  if (WHOLE) {
    if (tile >= w.tiles) return;
    cur = static_cast<int64_t>(tile) * w.blocks;
    rg.end = cur + w.blocks;
  }
  while (true) {
    const int64_t in_seq = cur - base;
    const int unit = static_cast<int>(in_seq / w.blocks);
    const int blk0 = static_cast<int>(in_seq - static_cast<int64_t>(unit) * w.blocks);
    const int nblk = static_cast<int>(min(static_cast<int64_t>(w.blocks - blk0), rg.end - cur));
    const int group = unit / w.tiles;
    const int h = group * p.team + cta % p.team;
    const int row0 = (unit - group * w.tiles) * C::kRows;
    const int rows = min(C::kRows, w.q_len * p.g - row0);      // of this tile

    const int tile_seen = seen_keys(p, w, (row0 + rows - 1) / p.g);

    // This warp's 16-key steps of the blocks: those that some row sees.
    const int key00 = blk0 * kRowKeys + warp_key;
    const int key_end = min(tile_seen, (blk0 + nblk) * kRowKeys);
    const int steps = key00 < key_end ? (key_end - key00 + step_keys - 1) >> (C::kStepLog2 + cshift) : 0;
    const int32_t* trow = p.table + b * p.table_stride;
    auto page_of = [&](int s) {
      if (s >= steps) return 0;
      // (a whole unit's first 32 pages are at hand: its blocks begin at key 0)
      const int pg = WHOLE && s < 32 ? (ahead >= 0 && ahead < p.pages ? ahead : -1)
                                     : page_at(trow, key00 + s * step_keys, p.page_shift,
                                               p.max_pages, p.pages);
      if (pg < 0) atomicMax(p.status, kDevBadPage);
      return pg;
    };
    int ids = page_of(lane), ids_next = page_of(32 + lane);
    const int64_t kh = (h * p.kc_h + crow * p.kc_r + cchunk * 8) * 2;
    const int64_t vh = (h * p.vc_h + crow * p.vc_r + cchunk * 8) * 2;
    const int64_t kstep = p.kc_r * (2 * RPI), vstep = p.vc_r * (2 * RPI);
    auto issue = [&](int s) {
      if (s < steps) {
        if (s > 0 && (s & 31) == 0) {
          ids = ids_next;
          ids_next = page_of(s + 32 + lane);
        }
        const int pg = __shfl_sync(0xffffffffu, ids, s & 31);
        const int key0 = key00 + s * step_keys;
        const int in = key0 & page_mask;
        const uint32_t st = ring + (s % C::kStages) * C::kStage;
        if (pg >= 0 && key0 + 16 <= w.kv_len && p.D == DT) {
          const char* ks = kc + kh + (pg * p.kc_p + in * p.kc_r) * 2;
          const char* vs = vc + vh + (pg * p.vc_p + in * p.vc_r) * 2;
#pragma unroll
          for (int it = 0; it < 16 / RPI; ++it) {
            const int r = it * RPI + crow;
            const uint32_t at = st + r * (DT * 2) + ((cchunk ^ (r & 7)) * 16);
            cp_async16(at, ks, 16);
            cp_async16(at + C::kTile, vs, 16);
            ks += kstep;
            vs += vstep;
          }
        } else {
          // The sequence's last keys, a page outside the cache, channels behind
          // D: zeros where there is nothing to copy.
          const int64_t pgc = pg < 0 ? 0 : pg;
          const char* ks = kc + kh + (pgc * p.kc_p + in * p.kc_r) * 2;
          const char* vs = vc + vh + (pgc * p.vc_p + in * p.vc_r) * 2;
          const int left = pg < 0 || !cin ? 0 : w.kv_len - key0 - crow;
#pragma unroll
          for (int it = 0; it < 16 / RPI; ++it) {
            const int r = it * RPI + crow;
            const uint32_t at = st + r * (DT * 2) + ((cchunk ^ (r & 7)) * 16);
            const bool in_seq = it * RPI < left;
            cp_async16(at, in_seq ? ks + it * kstep : kc, in_seq ? 16 : 0);
            cp_async16(at + C::kTile, in_seq ? vs + it * vstep : vc, in_seq ? 16 : 0);
          }
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < C::kStages - 1; ++s) issue(s);

    // Q fragments and what each of this thread's rows sees.
    uint32_t qf[MT][DT / 16][4];
    int lim[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int r = mt * 16 + hf * 8 + lane / 4;
        const bool in = r < rows;
        const int tok = (row0 + r) / p.g, hd = (row0 + r) - tok * p.g;
        lim[mt][hf] = in ? seen_keys(p, w, tok) : 0;
        const uint16_t* src = static_cast<const uint16_t*>(p.q) +
                              static_cast<int64_t>(w.begin + tok) * p.q_st +
                              static_cast<int64_t>(h * p.g + hd) * p.q_sh + (lane & 3) * 2;
#pragma unroll
        for (int kk = 0; kk < DT / 16; ++kk)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int d = kk * 16 + c * 8;
            qf[mt][kk][2 * c + hf] =
                in && d < p.D ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
          }
      }

    float m[MT][2], l[MT][2], o[MT][DT / 8][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      m[mt][0] = m[mt][1] = -INFINITY;
      l[mt][0] = l[mt][1] = 0.f;
#pragma unroll
      for (int n = 0; n < DT / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.f;
    }

    for (int s = 0; s < steps; ++s) {
      cp_async_wait<C::kStages - 2>();
      __syncwarp();
      issue(s + C::kStages - 1);
      const uint32_t st = ring + (s % C::kStages) * C::kStage;
      const int key0 = key00 + s * step_keys;
      // S = Q K^T for 16 keys: two 8-key column tiles.
      float sc[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[mt][n][e] = 0.f;
      {
        const int r = (lane >> 4) * 8 + (lane & 7);
        const uint32_t row = st + r * (DT * 2);
#pragma unroll
        for (int kk = 0; kk < DT / 16; ++kk) {
          uint32_t kf[4];
          ldsm4(row + (((kk * 2 + ((lane >> 3) & 1)) ^ (r & 7)) * 16), kf);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            if (mt * 16 >= rows) continue;
            mma_16816<F16>(sc[mt][0], qf[mt][kk], kf[0], kf[1]);
            mma_16816<F16>(sc[mt][1], qf[mt][kk], kf[2], kf[3]);
          }
        }
      }
      // Online softmax in the exp2 domain.  The reference maximum is raised
      // only when a row outgrows it by 2^8, which keeps rescales rare and the
      // weights within the 16-bit types' range; O / l is exact for any of them.
      uint32_t pf[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if (mt * 16 >= rows) continue;
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + n * 8 + (lane & 3) * 2 + (e & 1);
            float x = sc[mt][n][e] * p.scale_log2;
            if (key >= lim[mt][e >> 1]) x = -INFINITY;
            sc[mt][n][e] = x;
            mx[e >> 1] = fmaxf(mx[e >> 1], x);
          }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 1));
          mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 2));
        }
        if (__any_sync(0xffffffffu, mx[0] > m[mt][0] + 8.f || mx[1] > m[mt][1] + 8.f)) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const float mn = fmaxf(m[mt][hf], mx[hf]);
            const float al = mn == -INFINITY ? 1.f : ex2_approx(m[mt][hf] - mn);
            m[mt][hf] = mn;
            l[mt][hf] *= al;
#pragma unroll
            for (int n = 0; n < DT / 8; ++n) {
              o[mt][n][2 * hf] *= al;
              o[mt][n][2 * hf + 1] *= al;
            }
          }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const float ref = m[mt][hf] == -INFINITY ? 0.f : m[mt][hf];
            const float p0 = ex2_approx(sc[mt][n][2 * hf] - ref);
            const float p1 = ex2_approx(sc[mt][n][2 * hf + 1] - ref);
            l[mt][hf] += p0 + p1;
            pf[mt][2 * n + hf] = pack_16x2<F16>(p0, p1);
          }
      }
      // O += P V.
      {
        const int r = ((lane >> 3) & 1) * 8 + (lane & 7);
        const uint32_t row = st + C::kTile + r * (DT * 2);
#pragma unroll
        for (int nn = 0; nn < DT / 16; ++nn) {
          uint32_t vf[4];
          ldsm4_t(row + (((nn * 2 + (lane >> 4)) ^ (r & 7)) * 16), vf);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            if (mt * 16 >= rows) continue;
            mma_16816<F16>(o[mt][2 * nn], pf[mt], vf[0], vf[1]);
            mma_16816<F16>(o[mt][2 * nn + 1], pf[mt], vf[2], vf[3]);
          }
        }
      }
    }
    cp_async_wait<0>();

    // Join the warps: everything against the largest of their maxima.
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        l[mt][hf] += __shfl_xor_sync(0xffffffffu, l[mt][hf], 1);
        l[mt][hf] += __shfl_xor_sync(0xffffffffu, l[mt][hf], 2);
        if ((lane & 3) == 0) {
          const int r = mt * 16 + hf * 8 + lane / 4;
          s_m[warp * C::kRows + r] = m[mt][hf];
          s_l[warp * C::kRows + r] = l[mt][hf];
        }
      }
    __syncthreads();        // also: every warp is done with its ring
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int r = mt * 16 + hf * 8 + lane / 4;
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < C::kWarps; ++i) top = fmaxf(top, s_m[i * C::kRows + r]);
        const float al = m[mt][hf] == -INFINITY ? 0.f : ex2_approx(m[mt][hf] - top);
#pragma unroll
        for (int n = 0; n < DT / 8; ++n)
          *reinterpret_cast<float2*>(s_o + (warp * C::kRows + r) * DT + n * 8 + (lane & 3) * 2) =
              make_float2(o[mt][n][2 * hf] * al, o[mt][n][2 * hf + 1] * al);
      }
    __syncthreads();
    const bool first = blk0 == 0, last = blk0 + nblk == w.blocks;
    const bool shared = CUT == kWholeWide && cluster > 1;    // to add up in the cluster
    float* slot = shared ? reinterpret_cast<float*>(smem + C::kSumOff)
                         : p.part + static_cast<int64_t>(2 * cta + (first ? 1 : 0)) * C::kSlot;
    auto put = [&](int r, int d, const float4& acc, float sum) {
      if (d >= p.D) return;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int tok = (row0 + r) / p.g, hd = (row0 + r) - tok * p.g;
      uint16_t* dst = static_cast<uint16_t*>(p.o) + static_cast<int64_t>(w.begin + tok) * p.o_st +
                      static_cast<int64_t>(h * p.g + hd) * p.o_sh + d;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_16x2<F16>(acc.x * inv, acc.y * inv),
                                                  pack_16x2<F16>(acc.z * inv, acc.w * inv));
    };
    for (int i = threadIdx.x; i < rows * (DT / 4); i += C::kThreads) {
      const int r = i / (DT / 4), d = (i - r * (DT / 4)) * 4;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int k = 0; k < C::kWarps; ++k) top = fmaxf(top, s_m[k * C::kRows + r]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < C::kWarps; ++k) {
        const float mk = s_m[k * C::kRows + r];
        sum += mk == -INFINITY ? 0.f : s_l[k * C::kRows + r] * ex2_approx(mk - top);
        const float4 x = *reinterpret_cast<const float4*>(s_o + (k * C::kRows + r) * DT + d);
        acc.x += x.x;
        acc.y += x.y;
        acc.z += x.z;
        acc.w += x.w;
      }
      if (first && last && !shared) {
        put(r, d, acc, sum);
      } else {
        *reinterpret_cast<float4*>(slot + r * DT + d) = acc;
        if (d == 0) {
          slot[C::kRows * DT + r] = top;
          slot[C::kRows * DT + C::kRows + r] = sum;
        }
      }
    }
    if (shared) {
      cluster_sync();
      // The cluster's CTAs share the sums out, in the order of the ranks each.
      const uint32_t at = smem_u32(slot);
      for (int i = rank * C::kThreads + threadIdx.x; i < rows * (DT / 4);
           i += C::kThreads << cshift) {
        const int r = i / (DT / 4), d = (i - r * (DT / 4)) * 4;
        float m8[8], top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          m8[k] = k < cluster ? cluster_load(at + (C::kRows * DT + r) * 4, k) : -INFINITY;
          top = fmaxf(top, m8[k]);
        }
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (k >= cluster) continue;
          const float al = m8[k] == -INFINITY ? 0.f : ex2_approx(m8[k] - top);
          sum += cluster_load(at + (C::kRows * DT + C::kRows + r) * 4, k) * al;
          const float4 x = cluster_load4(at + (r * DT + d) * 4, k);
          acc.x += x.x * al;
          acc.y += x.y * al;
          acc.z += x.z * al;
          acc.w += x.w * al;
        }
        put(r, d, acc, sum);
      }
      cluster_sync();       // nobody's sums are read any more
    }
    cur += nblk;
    if (WHOLE) {
      tile += p.tile_ctas;
      if (tile >= w.tiles) break;
      cur = static_cast<int64_t>(tile) * w.blocks;
      rg.end = cur + w.blocks;
    } else if (cur >= rg.end) {
      // The unit that this CTA begins and others end, for the join.
      if (threadIdx.x == 0) {
        OpenUnit u = {0, h, row0, rows, w.begin};
        if (first && !last)
          u.parts = 1 + static_cast<int>((w.blocks - nblk + rg.per - 1) / rg.per);
        p.open[cta] = u;
      }
      break;
    }
    __syncthreads();        // the ring is free again
    if (!WHOLE && last && unit + 1 == w.tiles * (p.Hkv / p.team)) {
      base += weight(p, w);
      do {
        w = row_work(p, ++b, C::kRows);
      } while (w.tiles == 0);
    }
  }
}

// Adds up the parts of the unit that CTA blockIdx.x of the row kernel began and
// others ended.  A warp has the loads of kJoinAhead parts of a row in flight; of more
// parts the CTA's warps take a share each, and their sums are added in the warps'
// order.
constexpr int kJoinAhead = 8;
constexpr int kJoinRows = 8;            // CTAs over a unit's rows, at most
template <int DT, int MT, bool F16>
__global__ void __launch_bounds__(kRowThreads)
    paged_rows_join(const PagedParams p) {
  using C = RowCfg<DT, MT>;
  constexpr int E = DT / 32;            // channels of a lane
  __shared__ __align__(16) float s_acc[kRowWarps][DT];
  __shared__ float s_top[kRowWarps], s_sum[kRowWarps];
  grid_dependency_wait();
  const OpenUnit u = p.open[blockIdx.x];
  if (u.parts == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Part 0 is slot 1 of this CTA, part i slot 0 of its head's in the i-th team behind.
  auto slot = [&](int i) {
    return p.part +
           static_cast<int64_t>(2 * (blockIdx.x + i * p.team) + (i == 0 ? 1 : 0)) * C::kSlot;
  };
  float top, sum, acc[E];
  // Parts first, first + step, ... of row r.
  auto add = [&](int r, int first, int step) {
    top = -INFINITY;
    sum = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int i0 = first; i0 < u.parts; i0 += step * kJoinAhead) {
      float m[kJoinAhead], l[kJoinAhead], x[kJoinAhead][E];
#pragma unroll
      for (int k = 0; k < kJoinAhead; ++k) {
        const int i = i0 + k * step;
        const bool in = i < u.parts;
        const float* s = slot(in ? i : i0);
        m[k] = in ? s[C::kRows * DT + r] : -INFINITY;
        l[k] = s[C::kRows * DT + C::kRows + r];
        if constexpr (DT == 128) {
          const float4 v = *reinterpret_cast<const float4*>(s + r * DT + lane * 4);
          x[k][0] = v.x;
          x[k][1] = v.y;
          x[k][2] = v.z;
          x[k][3] = v.w;
        } else {
          const float2 v = *reinterpret_cast<const float2*>(s + r * DT + lane * 2);
          x[k][0] = v.x;
          x[k][1] = v.y;
        }
      }
      float now = top;
#pragma unroll
      for (int k = 0; k < kJoinAhead; ++k) now = fmaxf(now, m[k]);
      const float keep = top == -INFINITY ? 0.f : ex2_approx(top - now);
      sum *= keep;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= keep;
#pragma unroll
      for (int k = 0; k < kJoinAhead; ++k) {
        if (i0 + k * step >= u.parts) continue;
        // (a part that saw only scores that are no numbers has no maximum, but its O)
        const float al = m[k] == -INFINITY ? 0.f : ex2_approx(m[k] - now);
        sum += l[k] * al;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += x[k][e] * al;
      }
      top = now;
    }
  };
  auto row_out = [&](int r) {
    const int tok = (u.row0 + r) / p.g, hd = (u.row0 + r) - tok * p.g;
    return static_cast<uint16_t*>(p.o) + static_cast<int64_t>(u.begin + tok) * p.o_st +
           static_cast<int64_t>(u.h * p.g + hd) * p.o_sh;
  };
  if (u.parts <= kJoinAhead) {
    for (int r = blockIdx.y * kRowWarps + warp; r < u.rows; r += gridDim.y * kRowWarps) {
      add(r, 0, 1);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int e = 0; e < E; e += 2)
        if (lane * E < p.D)
          *reinterpret_cast<uint32_t*>(row_out(r) + lane * E + e) =
              pack_16x2<F16>(acc[e] * inv, acc[e + 1] * inv);
    }
    return;
  }
  for (int r = blockIdx.y; r < u.rows; r += gridDim.y) {
    add(r, warp, kRowWarps);
#pragma unroll
    for (int e = 0; e < E; ++e) s_acc[warp][lane * E + e] = acc[e];
    if (lane == 0) {
      s_top[warp] = top;
      s_sum[warp] = sum;
    }
    __syncthreads();
    const int d = threadIdx.x * 2;
    if (d < p.D) {
      float most = -INFINITY, total = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
      for (int k = 0; k < kRowWarps; ++k) most = fmaxf(most, s_top[k]);
#pragma unroll
      for (int k = 0; k < kRowWarps; ++k) {
        const float al = s_top[k] == -INFINITY ? 0.f : ex2_approx(s_top[k] - most);
        total += s_sum[k] * al;
        a0 += s_acc[k][d] * al;
        a1 += s_acc[k][d + 1] * al;
      }
      const float inv = total == 0.f ? 0.f : 1.f / total;
      *reinterpret_cast<uint32_t*>(row_out(r) + d) = pack_16x2<F16>(a0 * inv, a1 * inv);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
template <int DT, int MT, bool F16, Cut CUT>
int launch_rows_kernel(const PagedParams& p, cudaStream_t stream) {
  using C = RowCfg<DT, MT, CUT>;
  static KernelPrep prep;
  int dev = 0;
  const int rc = prepare_kernel(
      prep, reinterpret_cast<const void*>(paged_rows_kernel<DT, MT, F16, CUT>), C::kSmem, &dev);
  if (rc != FA_OK) return rc;
  return launch_after(paged_rows_kernel<DT, MT, F16, CUT>, dim3((p.ctas * p.team) << p.cluster_shift),
                      C::kThreads, C::kSmem, 1 << p.cluster_shift, stream, p);
}

template <int DT, int MT, bool F16>
int launch_rows(const PagedParams& p, Cut cut, int rows, cudaStream_t stream) {
  if (cut == kWhole) return launch_rows_kernel<DT, MT, F16, kWhole>(p, stream);
  if (MT == 1 && cut == kWholeWide) return launch_rows_kernel<DT, 1, F16, kWholeWide>(p, stream);
  const int rc = launch_rows_kernel<DT, MT, F16, kSplit>(p, stream);
  if (rc != FA_OK) return rc;
  return launch_after(paged_rows_join<DT, MT, F16>,
                      dim3(p.ctas * p.team, rows < kJoinRows ? rows : kJoinRows), kRowThreads, 0, 1,
                      stream, p);
}

template <int DT, int MT>
int launch_rows_t(const PagedParams& p, bool f16, Cut cut, int rows, cudaStream_t stream) {
  return f16 ? launch_rows<DT, MT, true>(p, cut, rows, stream)
             : launch_rows<DT, MT, false>(p, cut, rows, stream);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Strides of `n` dimensions: multiples of 8 elements where the dimension has
// more than one entry, not negative, and not 0 where written.
bool strides_ok(const int64_t* st, const int64_t* sizes, int n, bool written) {
  for (int i = 0; i < n; ++i)
    if (sizes[i] > 1 && (st[i] < (written ? 1 : 0) || st[i] % 8 != 0)) return false;
  return true;
}

// The scale of the exponent to base 2, as the kernels have it.
float scale_log2(const fa_paged_attn_args* a) {
  return static_cast<float>(a->scale * 1.4426950408889634);
}

int check_paged_attn(const fa_paged_attn_args* a) {
  constexpr int64_t kMax = 0x7fffffffLL, kMaxPlaces = kMax - 4096;
  if (!a || !a->q || !a->o || !a->k_cache || !a->v_cache || !a->block_table || !a->kv_lens)
    return FA_ERR_NULL;
  if (a->dtype != FA_BF16 && a->dtype != FA_F16) return FA_ERR_ARG;
  if (a->T <= 0 || a->B <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->T > kMax || a->B >= kMax ||
      a->Hkv > 65536 || a->Hq > 65536 || a->Hq % a->Hkv || a->Hq / a->Hkv > 128 ||
      a->T * a->Hq > kMax || a->max_q_len <= 0)
    return FA_ERR_SHAPE;
  if (!a->cu_seqlens && a->T != a->B) return FA_ERR_SHAPE;
  if (a->D < 8 || a->D > 128 || a->D % 8) return FA_ERR_HEAD_DIM;
  if (!std::isfinite(scale_log2(a))) return FA_ERR_ARG;
  if (a->pages <= 0 || a->pages > kMax || a->max_pages <= 0 || a->max_pages > kMax ||
      a->page_size < 16 || a->page_size > 1024 || (a->page_size & (a->page_size - 1)) ||
      a->max_pages * a->page_size > kMaxPlaces)
    return FA_ERR_SHAPE;
  if (a->B > 1 && a->table_stride < a->max_pages) return FA_ERR_STRIDE;
  const int64_t qs[2] = {a->T, a->Hq}, cs[3] = {a->pages, a->page_size, a->Hkv};
  if (!strides_ok(a->q_strides, qs, 2, false) || !strides_ok(a->o_strides, qs, 2, true) ||
      !strides_ok(a->k_cache_strides, cs, 3, false) ||
      !strides_ok(a->v_cache_strides, cs, 3, false) || !aligned16(a->q) || !aligned16(a->o) ||
      !aligned16(a->k_cache) || !aligned16(a->v_cache))
    return FA_ERR_ALIGN;
  return FA_OK;
}

// Which kernel runs, by sizes that the host knows.
//  * Few rows: the row kernel with a cluster per sequence, head and 16 rows, of
//    CTAs of 16 warps (8 with D > 64), as many as get 2 steps or more of their own
//    and leave a CTA per SM, up to 8 steps of each.  37 tokens over 1061 keys, 16
//    heads of 64: 9.4 us, 16.5 split and joined, 21 by the tile kernel.  8 sequences
//    of up to 2000 keys, 32/8 heads of 128: 12.3 us, split 14.8; 2 of up to 8192
//    (16 steps): 18.2, split 13.1.
//  * Over up to 1024 keys again no join: a CTA per sequence, head and 32 rows, for
//    sequences of up to kRowMax rows (256 sequences of 512 keys, 8 heads of 64: 36
//    us, split 51) and for calls of up to kWholeWork operations over the whole
//    table (28 sequences of up to 30 tokens over 73 keys, 24/2 heads of 80: 11.4 us,
//    15.7 by the tile kernel, 33.6 split; 5 of up to 188 tokens, 32/2 heads of 96,
//    above it: 25, 16.8 by the tile kernel).
//  * Split and joined, the row kernel takes the other sequences of up to kRowMax
//    rows (single tokens), and chunks of up to kRowWork operations, where the tile
//    kernel's plan and join cost more than its products save.
//  * The tile kernel takes chunks, and then the batch's short sequences too: a
//    second launch for those costs more than a tile kernel's unit of one token.
constexpr int kRowMax = 32;
constexpr double kRowWork = 1e8, kWholeWork = 1e9;

// Clusters of 1 << shift CTAs of the wide row kernel that device dev holds at
// once (clusters lie within one of its parts: 16 of 8 CTAs do not fit 148 SMs).
int max_clusters(int dev, bool narrow, int shift) {
  static std::atomic<int> known[64][2][4];
  if (dev < 0 || dev >= 64) return 0;
  std::atomic<int>& slot = known[dev][narrow ? 1 : 0][shift];
  int n = slot.load(std::memory_order_relaxed);
  if (n > 0) return n;
  const void* kern = narrow ? reinterpret_cast<const void*>(paged_rows_kernel<64, 1, false, kWholeWide>)
                            : reinterpret_cast<const void*>(paged_rows_kernel<128, 1, false, kWholeWide>);
  const int smem = narrow ? RowCfg<64, 1, kWholeWide>::kSmem : RowCfg<128, 1, kWholeWide>::kSmem;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(8 * 148);
  cfg.blockDim = dim3(narrow ? RowCfg<64, 1, kWholeWide>::kThreads
                             : RowCfg<128, 1, kWholeWide>::kThreads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 1 << shift;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
    (void)cudaGetLastError();
    return 0;
  }
  slot.store(n, std::memory_order_relaxed);
  return n;
}

struct Choice {
  bool tiles;
  bool rows32;          // row tiles of 32 rows, else 16
  Cut cut;
  int tile_ctas;        // whole units: CTAs over a head's row tiles
  int cluster_shift;    // and CTAs of each: 1 << this
};

Choice choose(const fa_paged_attn_args* a, int dev, int sms) {
  const int64_t longest = (a->max_q_len < a->T ? a->max_q_len : a->T) * (a->Hq / a->Hkv);
  const int64_t keys = a->max_pages * a->page_size, units = a->B * a->Hkv;
  const int64_t tiles16 = (longest + 15) / 16, tiles32 = (longest + 31) / 32;
  const int step = a->D <= 64 ? RowCfg<64, 1, kWholeWide>::kStep : RowCfg<128, 1, kWholeWide>::kStep;
  if (units <= sms && units * tiles16 <= sms) {
    int shift = 0;
    while (shift < 3 && keys > (2ll << shift) * step &&
           units * tiles16 <= max_clusters(dev, a->D <= 64, shift + 1))
      ++shift;
    if (keys <= 8 * (static_cast<int64_t>(step) << shift))
      return {false, false, kWholeWide, static_cast<int>(tiles16), shift};
  }
  const double most = 4.0 * a->T * a->Hq * a->D * keys;
  if (keys <= 1024 && (longest <= kRowMax || most <= kWholeWork) && units <= 0x7fffffffLL / tiles32)
    return {false, longest > 16, kWhole, static_cast<int>(tiles32), 0};
  // The tile kernel's copies need real strides; it masks scores before it scales them
  // and takes the maximum before, so its scale has to keep their order and -infinity.
  const bool flat = (a->q_strides[0] == 0 && a->T > 1) || (a->q_strides[1] == 0 && a->Hq > 1) ||
                    (a->k_cache_strides[0] == 0 && a->pages > 1) || a->k_cache_strides[1] == 0 ||
                    (a->k_cache_strides[2] == 0 && a->Hkv > 1) ||
                    (a->v_cache_strides[0] == 0 && a->pages > 1) || a->v_cache_strides[1] == 0 ||
                    (a->v_cache_strides[2] == 0 && a->Hkv > 1);
  const bool ordered = scale_log2(a) > 0.f;
  return {longest > kRowMax && most > kRowWork && !flat && ordered, longest > 16, kSplit, 1, 0};
}

// Teams of the row kernel: of the size, up to 16 heads, that fills the device
// best, and as many as it holds at once.
struct Teams {
  int heads, count;
};
Teams row_teams(const fa_paged_attn_args* a, const Choice& c, int sms) {
  if (c.cut != kSplit) return {static_cast<int>(a->Hkv), static_cast<int>(a->B) * c.tile_ctas};
  const int ctas = sms * (c.rows32 ? (a->D <= 64 ? RowCfg<64, 2>::kCtasPerSm
                                                 : RowCfg<128, 2>::kCtasPerSm)
                                   : (a->D <= 64 ? RowCfg<64, 1>::kCtasPerSm
                                                 : RowCfg<128, 1>::kCtasPerSm));
  Teams best = {1, ctas};
  for (int n = 2; n <= 16; ++n)
    if (a->Hkv % n == 0 && ctas / n * n >= best.heads * best.count * 0.97) best = {n, ctas / n};
  return best;
}

// A CTA's parts of units: of the one that its range begins in and of the last.
int64_t part_bytes(const fa_paged_attn_args* a, const Choice& c) {
  return 2 * (c.rows32 ? 32 : 16) * ((a->D <= 64 ? 64 : 128) + 2) * 4;
}

}  // namespace
}  // namespace fa

extern "C" int64_t fa_paged_attn_workspace(const fa_paged_attn_args* a) {
  using namespace fa;
  const int rc = check_paged_attn(a);
  if (rc != FA_OK) return -rc;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -FA_ERR_CUDA;
  const int sms = sm_count(dev);
  if (sms <= 0) return -FA_ERR_CUDA;
  const Choice c = choose(a, dev, sms);
  if (c.tiles) return paged_tiles_bytes(a, sms);
  if (c.cut != kSplit) return 0;
  const Teams t = row_teams(a, c, sms);
  return t.heads * t.count * (static_cast<int64_t>(sizeof(OpenUnit)) + part_bytes(a, c));
}

extern "C" int fa_paged_attn(const fa_paged_attn_args* a, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  using namespace fa;
  int rc = check_paged_attn(a);
  if (rc != FA_OK) return rc;
  int dev = 0;
  if ((rc = prepare_device(nullptr, 0, &dev)) != FA_OK) return rc;
  const int64_t need = fa_paged_attn_workspace(a);
  if (need < 0) return static_cast<int>(-need);
  if (need > 0 && (!workspace || workspace_bytes < need)) return FA_ERR_WORKSPACE;
  if (!aligned16(workspace)) return FA_ERR_ALIGN;
  PagedParams p = {};
  p.q = a->q;
  p.o = a->o;
  p.kc = a->k_cache;
  p.vc = a->v_cache;
  p.table = a->block_table;
  p.lens = a->kv_lens;
  p.cu = a->cu_seqlens;
  p.q_st = a->q_strides[0];
  p.q_sh = a->q_strides[1];
  p.o_st = a->o_strides[0];
  p.o_sh = a->o_strides[1];
  p.kc_p = a->k_cache_strides[0];
  p.kc_r = a->k_cache_strides[1];
  p.kc_h = a->k_cache_strides[2];
  p.vc_p = a->v_cache_strides[0];
  p.vc_r = a->v_cache_strides[1];
  p.vc_h = a->v_cache_strides[2];
  p.table_stride = a->table_stride;
  p.T = static_cast<int>(a->T);
  p.B = static_cast<int>(a->B);
  p.Hkv = static_cast<int>(a->Hkv);
  p.g = static_cast<int>(a->Hq / a->Hkv);
  p.D = static_cast<int>(a->D);
  p.pages = static_cast<int>(a->pages);
  p.page_shift = __builtin_ctzll(static_cast<unsigned long long>(a->page_size));
  p.max_pages = static_cast<int>(a->max_pages);
  p.causal = a->causal != 0;
  p.scale_log2 = scale_log2(a);
  p.status = device_status_ptr();
  if (p.status == nullptr) return FA_ERR_CUDA;
  const int sms = sm_count(dev);
  const bool f16 = a->dtype == FA_F16;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Choice c = choose(a, dev, sms);
  if (c.tiles) {
    p.ctas = sms;
    return launch_paged_tiles(a, p, workspace, s);
  }
  const Teams t = row_teams(a, c, sms);
  p.ctas = t.count;
  p.team = t.heads;
  p.tile_ctas = c.tile_ctas;
  p.cluster_shift = c.cluster_shift;
  p.part = static_cast<float*>(workspace);
  p.open = reinterpret_cast<OpenUnit*>(static_cast<char*>(workspace) +
                                       t.heads * t.count * part_bytes(a, c));
  p.min_blocks = 4;
  // (the join's CTAs go over more rows than these where max_q_len was too small)
  const int64_t longest = (a->max_q_len < a->T ? a->max_q_len : a->T) * p.g;
  const int rows = static_cast<int>(longest < 32 ? longest : 32);
  if (c.rows32)
    return p.D <= 64 ? launch_rows_t<64, 2>(p, f16, c.cut, rows, s)
                     : launch_rows_t<128, 2>(p, f16, c.cut, rows, s);
  return p.D <= 64 ? launch_rows_t<64, 1>(p, f16, c.cut, rows, s)
                   : launch_rows_t<128, 1>(p, f16, c.cut, rows, s);
}
