// The tensor-core kernel of the paged attention, for chunks of new tokens.
//
// A tile is 128 rows of one (sequence, key head): floor(128 / g) consecutive new
// tokens with their g query heads, token by token (g = Hq / Hkv), so the heads
// that share a key head share its loads and one tile serves any group.  A unit
// is two tiles; per 128 keys the tensor core computes, in this order,
//   O_0 += P_0(j-1) V_{j-1};  S_0 = Q_0 K_j^T;  O_1 += P_1(j-1) V_{j-1};  S_1 = Q_1 K_j^T
// so one tile's products run while the other's softmax does.  Warp roles (384
// threads, one CTA per SM):
//   warps 0-3, 4-7  softmax of tile 0 and 1 (a thread = a row = a TMEM lane)
//   warp 8          loads: Q tiles once per unit, K by pages into a ring
//   warp 9          TMEM allocation and the single thread that issues tcgen05.mma
//   warp 10         loads V by pages into the ring
// S_t lives in TMEM columns [128 t, 128 t + 128), P_t over its first half as 16-bit
// pairs, O_t at 256 + D t.
//
// Bound by the power limit and by the chain S -> softmax -> P of each tile: 2800
// clocks per 128 keys for 2048 clocks of tensor work (D = 128).  512 tokens over
// 32768 keys, 32/8 heads of 128: 217 to 223 us, 1240 TFLOP/s, the tensor pipe 72 %
// active at 1.56 GHz; a causal prompt of 8192 tokens, 32 heads of 128: 433 to 443 us,
// 1255 TFLOP/s.  After a tenth of a second of nothing else the power limit takes the
// clock further down: 256 and 506 us.  With D = 64 the softmax alone takes the 2800
// clocks (half the issue slots, 58 % of the exponential unit), 178 us and 766
// TFLOP/s for that chunk: room for P beside S, so that S comes a block ahead, did not
// change an earlier 223 us (232), and four tiles of 64 keys took 191 for 203, but 131
// for 114 over shorter lists.
//
// P is rounded to the 16-bit type that the matrix instruction takes, while the sum l
// adds the unrounded weights, in fp32 like O; fp16 weights below 2^-24 of the row's
// reference vanish from P.  The outputs' error against fp64 is 0.0023 of their size in
// bf16 and 0.00029 in fp16, where fp32 arithmetic rounded once has 0.0017 and 0.00021.
//
// Pages: a load box is min(page_size, 128) rows of one page, so a 128-key tile
// takes 128 / page_size boxes whose pages come from the block table, one lane of
// the loading warp per page.  Boxes behind the sequence's last key are not loaded;
// rows of V behind it are zeroed in shared memory, because 0 * NaN of a slot that
// was never written would reach the output.
//
// Work (decided on the device by paged_plan_kernel, from the lengths):
//  * whole units: CTAs take them from a counter, heads in groups whose K and V
//    fit half the L2, longest units first.  Of more than 4 units per SM, one that
//    is longer than a CTA's even share is cut into parts that go first.
//  * cut units, where there are up to 4 per SM and whole ones would leave CTAs
//    idle for longer than the parts cost: every CTA gets the same number of key
//    blocks, L.  A unit of more than L is cut at L, 2 L, ... and each such part is
//    one CTA's work; what is left of it, and shorter units, are laid end to end and
//    cut into equal ranges for the other CTAs.  The parts of one head's units begin
//    at the same keys, so the CTAs that read them run side by side in the L2: with
//    plain equal ranges 512 tokens over 32768 keys (8 key heads of 128) read the
//    cache from DRAM once for each of a head's 8 units (244 us against 221).
// A unit's parts leave (m, l, O) in the workspace and paged_tiles_join adds them
// in the order of the keys.
// Results depend on the lengths alone, never on timing.
#include <cuda_bf16.h>

#include <climits>

#include "paged_attn.h"
#include "sm100_tmem_wide.cuh"

namespace fa {
namespace {

constexpr int kRows = 128;           // rows of a tile (TMEM lanes)
constexpr int kKeys = 128;           // keys of a block
constexpr int kThreads = 384;
constexpr int kRegsCtrl = 72, kRegsSoftmax = 216;
static_assert(128 * kRegsCtrl + 256 * kRegsSoftmax <= 384 * 168,
              "the register split exceeds the launch's pool");
constexpr int kUnitsPerSm = 4;       // from here on only outliers are cut
constexpr int kPlanThreads = 640;       // at least the units that may be split
constexpr int kStartCells = 2;          // what a part's start and end cost, in key blocks
constexpr int kJoinCells = 8;           // what cutting costs the whole, in key blocks
constexpr int64_t kGroupBytes = 32ll << 20;   // K and V of the heads worked on at once

// A unit, or the part of one that a CTA computes.
struct Piece {
  int b, h;
  int tok0;              // the unit's first token within the sequence
  int q_begin, q_len, kv_len;
  int blk0;              // first key block
  int nt[2];             // key blocks of each tile from there (0: it sees none of them)
  int slot;              // where its part goes, -1: the whole unit
  int place0;            // the sequence's first new token's place
  int pad;
};
static_assert(sizeof(Piece) == 48, "pieces are copied as three 16-byte words");

// A unit in parts, for the join.
struct JoinUnit {
  int slot0, parts;
  int tok0, q_begin, q_len, h;
  int pad[2];
};
static_assert(sizeof(JoinUnit) == 32, "read as two 16-byte words");

// The plan, at the workspace's start.
enum : int { kSplit = 0, kJoins = 1, kNext = 2, kUnits = 3, kPieces = 4, kLongest = 5, kHeader = 8 };
struct TileParams : PagedParams {
  int tq;                // tokens of a tile
  int box_rows;          // rows of a load box
  int min_cells;         // least key blocks of a CTA's range
  int split_units;       // units from which on only outliers are cut
  int* plan;             // header
  int* prefix;           // [B + 1]: units (per head) of the sequences before
  int* first;            // [ctas + 1]: first piece of each CTA
  JoinUnit* join;        // [ctas]
  Piece* pieces;
};

struct PlanOffsets {
  int64_t prefix, first, join, pieces, parts, bytes;
};

__host__ __device__ constexpr int64_t up128(int64_t n) { return (n + 127) / 128 * 128; }

// ---------------------------------------------------------------------------
// Work
// ---------------------------------------------------------------------------
__device__ __forceinline__ int units_of(const TileParams& p, const SeqWork& w) {
  return (w.q_len + 2 * p.tq - 1) / (2 * p.tq);
}
// Key blocks that the tokens [tok0, tok0 + n) of the sequence see.
__device__ __forceinline__ int blocks_of(const TileParams& p, const SeqWork& w, int tok0, int n) {
  if (tok0 >= w.q_len) return 0;
  const int seen = seen_keys(p, w, min(tok0 + n, w.q_len) - 1);
  return (seen + kKeys - 1) / kKeys;
}
__device__ __forceinline__ Piece make_piece(const TileParams& p, const SeqWork& w, int b, int h,
                                            int u, int blk0, int blk1, int slot) {
  Piece x;
  x.b = b;
  x.h = h;
  x.tok0 = u * 2 * p.tq;
  x.q_begin = w.begin;
  x.q_len = w.q_len;
  x.kv_len = w.kv_len;
  x.blk0 = blk0;
#pragma unroll
  for (int t = 0; t < 2; ++t)
    x.nt[t] = max(0, min(blocks_of(p, w, x.tok0 + t * p.tq, p.tq), blk1) - blk0);
  x.slot = slot;
  x.place0 = w.place0;
  x.pad = 0;
  return x;
}
__device__ __forceinline__ void put_piece(Piece* to, const Piece& x) {
  int4* d = reinterpret_cast<int4*>(to);
  d[0] = make_int4(x.b, x.h, x.tok0, x.q_begin);
  d[1] = make_int4(x.q_len, x.kv_len, x.blk0, x.nt[0]);
  d[2] = make_int4(x.nt[1], x.slot, x.place0, 0);
}
__device__ __forceinline__ void put_join(JoinUnit* to, int slot0, int parts, int tok0,
                                         const SeqWork& w, int h) {
  int4* d = reinterpret_cast<int4*>(to);
  d[0] = make_int4(slot0, parts, tok0, w.begin);
  d[1] = make_int4(w.q_len, h, 0, 0);
}
// The sequence whose units (times heads) hold unit i.
template <typename I>
__device__ __forceinline__ int seq_of_unit(const int* prefix, int B, I heads, I i) {
  int lo = 0, hi = B;                   // prefix[lo] * heads <= i < prefix[hi] * heads
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] * heads <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}
// Unit i of the whole list: sequences in order, a sequence's heads in groups
// that stay in the L2, in a group the longest units (the last tokens) first.
__device__ __forceinline__ Piece whole_unit(const TileParams& p, int64_t i) {
  const int b = seq_of_unit<int64_t>(p.prefix, p.B, p.Hkv, i);
  const SeqWork w = seq_work(p, b);
  const int nu = p.prefix[b + 1] - p.prefix[b];
  const int r = static_cast<int>(i - static_cast<int64_t>(p.prefix[b]) * p.Hkv);
  const int64_t head_bytes = static_cast<int64_t>(max(1, w.kv_len)) * p.D * 4;
  const int fit = static_cast<int>(max(int64_t{1}, min(int64_t{p.Hkv}, kGroupBytes / head_bytes)));
  const int groups = (p.Hkv + fit - 1) / fit;
  const int hg = (p.Hkv + groups - 1) / groups;      // heads of a group, spread evenly
  const int g = r / (hg * nu);
  const int in = r - g * hg * nu;
  const int here = min(hg, p.Hkv - g * hg);
  const int u = nu - 1 - in / here;
  return make_piece(p, w, b, g * hg + in % here, u, 0, INT_MAX, -1);
}

// Exclusive prefix sum over the CTA's threads; *total: the sum.
__device__ __forceinline__ unsigned plan_scan(unsigned v, unsigned* red, unsigned* total) {
  constexpr int kWarps = kPlanThreads / 32;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  unsigned x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) red[w] = x;
  __syncthreads();
  unsigned y = lane < kWarps ? red[lane] : 0;     // every warp scans the warps' sums
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) y += z;
  }
  *total = __shfl_sync(0xffffffffu, y, 31);
  const unsigned before = __shfl_sync(0xffffffffu, y, w > 0 ? w - 1 : 0);
  return (w > 0 ? before : 0) + x - v;
}

// A unit of nb key blocks in parts of L: whole parts and what is left.
struct Parts {
  int whole, left;
};
__device__ __forceinline__ Parts cut_unit(int nb, int L) {
  Parts c = {0, nb};
  if (nb > L) {
    c.whole = static_cast<int>(static_cast<unsigned>(nb) / static_cast<unsigned>(L));
    c.left = nb - c.whole * L;
  }
  return c;
}
// Cells that the rest of a unit takes in the laid-out row of such rests.
__device__ __forceinline__ int rest_cells(const Parts& c) {
  return c.left > 0 || c.whole == 0 ? c.left + kStartCells : 0;
}

// One CTA.  Counts every sequence's units; where they are few, cuts their key
// blocks into the CTAs' shares.  Everything waits for it (6000 clocks, of which
// each of its prefix sums takes 400), so what it looks up again stays in shared
// memory and its numbers are packed into 32 bits.
constexpr int kMaxSplitCells = 1 << 23;       // of a batch that is cut up
constexpr int kMaxSplitCtas = 255;
__global__ void __launch_bounds__(kPlanThreads)
    paged_plan_kernel(const TileParams p) {
  __shared__ unsigned red[32];
  __shared__ int s_blocks[kPlanThreads];                // of (sequence, unit) pairs, one head
  __shared__ int s_prefix[kPlanThreads + 1];
  __shared__ SeqWork s_work[kPlanThreads];
  __shared__ unsigned long long s_all;
  __shared__ unsigned s_fits;
  __shared__ int s_longest, s_joins, s_pieces;
  grid_dependency_wait();
  grid_dependents_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    s_all = 0;
    s_fits = 0;
    s_longest = s_joins = s_pieces = 0;
  }
  unsigned pairs = 0;                   // (T and B are below 2^31, and so are units)
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    SeqWork w = {};
    if (b < p.B) w = seq_work(p, b);
    unsigned sum;
    const unsigned before = pairs + plan_scan(units_of(p, w), red, &sum);
    if (b < p.B) p.prefix[b] = static_cast<int>(before);
    if (b0 == 0) {
      s_prefix[tid] = static_cast<int>(before);
      s_work[tid] = w;
    }
    pairs += sum;
  }
  if (tid == 0) {
    p.prefix[p.B] = static_cast<int>(pairs);
    p.plan[kUnits] = static_cast<int>(pairs * p.Hkv);
    p.plan[kNext] = 0;
    if (p.B <= kPlanThreads) s_prefix[p.B] = static_cast<int>(pairs);
  }
  const uint64_t units64 = static_cast<uint64_t>(pairs) * p.Hkv;
  const bool few = units64 < static_cast<uint64_t>(p.split_units);   // (at most kPlanThreads)
  const bool held = p.B <= kPlanThreads;
  const int* prefix = held ? s_prefix : p.prefix;
  auto work = [&](int b) { return held ? s_work[b] : seq_work(p, b); };
  auto blocks_of_pair = [&](int i) {
    const int b = seq_of_unit(prefix, p.B, 1, i);
    return blocks_of(p, work(b), (i - prefix[b]) * 2 * p.tq, 2 * p.tq);
  };
  __syncthreads();
  // All units' cells (key blocks and kStartCells) and the longest unit.
  {
    uint64_t sum = 0;
    int longest = 0;
    for (int i = tid; i < static_cast<int>(pairs); i += kPlanThreads) {
      const int nb = blocks_of_pair(i);
      if (i < kPlanThreads) s_blocks[i] = nb;
      sum += nb + kStartCells;
      longest = max(longest, nb);
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      atomicAdd(&s_all, static_cast<unsigned long long>(sum));
      atomicMax(&s_longest, longest);
    }
  }
  __syncthreads();
  const uint64_t all64 = s_all * static_cast<uint64_t>(p.Hkv);
  const int longest = s_longest;
  const int units = static_cast<int>(units64);

  // The least cells of a CTA, of 20 tried, with which cut units fit the CTAs: a
  // warp tries one.
  const bool can_cut = few && all64 < kMaxSplitCells;
  const unsigned all = static_cast<unsigned>(all64);
  const int least =
      can_cut ? max(p.min_cells + kStartCells, static_cast<int>((all + p.ctas - 1) / p.ctas)) : 0;
  auto tried = [&](int j) { return least + (least * j + 39) / 40; };
  if (can_cut) {
    const int cells = tried(warp);
    unsigned whole = 0, rest = 0;
    for (int i = lane; i < static_cast<int>(pairs); i += 32) {
      const Parts c = cut_unit(s_blocks[i], cells - kStartCells);
      whole += c.whole;
      rest += rest_cells(c);
    }
    whole = __reduce_add_sync(0xffffffffu, whole);
    rest = __reduce_add_sync(0xffffffffu, rest);
    if (lane == 0 && whole * p.Hkv + (rest * p.Hkv + cells - 1) / cells <= p.ctas)
      atomicOr(&s_fits, 1u << warp);
  }
  __syncthreads();
  // (2 * least always fits: a part's start is a third of it at most)
  const int cells = s_fits ? tried(__ffs(s_fits) - 1) : 2 * least;
  const int L = cells - kStartCells;
  // Whole units end about a sixth of the longest after their even share, and not
  // before the longest; cut ones after their share and the join.
  const int end_whole =
      max(longest + kStartCells, units <= p.ctas ? 0 : least + longest / 6);
  const bool split = can_cut && cells + kJoinCells < end_whole;
  if (!split) {
    // A share's length for outliers; none is cut among few units.
    const uint64_t share = few ? static_cast<uint64_t>(INT_MAX)
                               : max(static_cast<uint64_t>(p.min_cells), all64 / p.ctas);
    const int most = p.split_units > 0 && share < INT_MAX ? static_cast<int>(share) : INT_MAX;
    if (longest > most) {
      for (int i = tid; i < static_cast<int>(pairs); i += kPlanThreads) {
        const int nb = blocks_of_pair(i);
        if (nb <= most) continue;
        const int b = seq_of_unit(prefix, p.B, 1, i);
        const SeqWork w = work(b);
        const int parts = (nb + most - 1) / most, len = (nb + parts - 1) / parts;
        const int join0 = atomicAdd(&s_joins, p.Hkv), piece0 = atomicAdd(&s_pieces, parts * p.Hkv);
        for (int h = 0; h < p.Hkv; ++h) {
          put_join(p.join + join0 + h, piece0 + h * parts, parts, (i - prefix[b]) * 2 * p.tq, w, h);
          for (int k = 0; k < parts; ++k)
            put_piece(p.pieces + piece0 + h * parts + k,
                      make_piece(p, w, b, h, i - prefix[b], k * len, min(nb, (k + 1) * len),
                                 piece0 + h * parts + k));
        }
      }
      __syncthreads();
    }
    if (tid == 0) {
      p.plan[kSplit] = 0;
      p.plan[kJoins] = s_joins;
      p.plan[kPieces] = s_pieces;
      p.plan[kLongest] = most;
    }
    return;
  }

  // Units in the order (sequence, head, unit).
  int b = 0, h = 0, u = 0;
  SeqWork w = {};
  Parts cut = {0, 0};
  int rest = 0;
  if (tid < units) {
    b = seq_of_unit(prefix, p.B, p.Hkv, tid);
    w = work(b);
    const unsigned nu = prefix[b + 1] - prefix[b];
    const unsigned r = tid - prefix[b] * p.Hkv;
    h = r / nu;
    u = r - h * nu;
    cut = cut_unit(s_blocks[prefix[b] + u], L);
    rest = rest_cells(cut);
  }
  // CTAs of the whole parts before this unit's, cells of the rests before it.
  unsigned total;
  unsigned before = plan_scan(static_cast<unsigned>(cut.whole) * kMaxSplitCells + rest, red, &total);
  const int cta0 = before / kMaxSplitCells, ctas_whole = total / kMaxSplitCells;
  const int ctas_rest = (total % kMaxSplitCells + cells - 1) / cells;
  const int at = before % kMaxSplitCells + kStartCells, end = at + cut.left;   // the rest's blocks
  int c0 = 0, n = 0;                                    // CTAs of the rest (a unit without keys:
  if (rest > 0) {                                       // where its start lies)
    c0 = static_cast<unsigned>(end > at ? at : at - 1) / static_cast<unsigned>(cells);
    n = end > at ? static_cast<unsigned>(end - 1) / static_cast<unsigned>(cells) - c0 + 1 : 1;
  }
  const int parts = cut.whole + n;
  const bool alone = parts <= 1;
  // Pieces of the rests before this unit's, slots, units in parts (1024, 2048, 1024 at most).
  before = plan_scan(n + (alone ? 0u : parts << 10 | 1u << 21), red, &total);
  const int piece0 = ctas_whole + (before & 1023), slot0 = before >> 10 & 2047;
  const int pieces = ctas_whole + (total & 1023);
  for (int i = 0; i < cut.whole; ++i) {
    put_piece(p.pieces + cta0 + i,
              make_piece(p, w, b, h, u, i * L, (i + 1) * L, alone ? -1 : slot0 + i));
    p.first[cta0 + i] = cta0 + i;
  }
  for (int i = 0; i < n; ++i) {
    const int lo = max(at, (c0 + i) * cells), hi = min(end, (c0 + i + 1) * cells);
    const int blk = cut.whole * L - at;
    put_piece(p.pieces + piece0 + i,
              make_piece(p, w, b, h, u, end > at ? blk + lo : 0, end > at ? blk + hi : 0,
                         alone ? -1 : slot0 + cut.whole + i));
    // The first piece of a CTA: one that goes on from the CTA before, or whose
    // unit is the first to have a key block (or its end) among the CTA's cells.
    const int unit_at = at - kStartCells;
    if (i > 0 || unit_at == 0 ||
        static_cast<unsigned>(unit_at - 1) / static_cast<unsigned>(cells) <
            static_cast<unsigned>(c0))
      p.first[ctas_whole + c0 + i] = piece0 + i;
  }
  if (!alone) put_join(p.join + (before >> 21), slot0, parts, u * 2 * p.tq, w, h);
  if (tid == 0) {
    p.plan[kSplit] = 1;
    p.plan[kJoins] = total >> 21;
  }
  if (tid <= p.ctas && tid >= ctas_whole + ctas_rest) p.first[tid] = pieces;
}

// ---------------------------------------------------------------------------
// Exponentials: a quarter of them on the FMA pipe
// ---------------------------------------------------------------------------
// The largest of two or three; NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x for two values: x = j + f with j the nearest whole number (the addition of
// 1.5 * 2^23 + 127 leaves j + 127 in the low mantissa bits), 2^f by the degree-3
// minimax polynomial of fit_exp2_poly.py (relative error 7.5e-5), times 2^j made of
// those bits.  x is held at -127, where 2^j is 0: a masked score weighs exactly
// nothing, whatever finite value it would multiply.  (Adding j to the exponent
// instead saves a product of every 2 values, but can give no less than 2^-125.)
// NaN, which an infinite score less an infinite reference is, stays NaN.
__device__ __forceinline__ void exp2_pair(float x0, float x1, float& r0, float& r1) {
  const uint64_t x = f2_pack(max_nan(x0, -127.f), max_nan(x1, -127.f));
  const uint64_t t = fadd2(x, f2_pack(12583039.f, 12583039.f));
  const uint64_t j = fadd2(t, f2_pack(-12583039.f, -12583039.f));
  const uint64_t f = ffma2(j, f2_pack(-1.f, -1.f), x);
  uint64_t q = ffma2(f2_pack(0.0551716685295105f, 0.0551716685295105f), f,
                     f2_pack(0.2426111251115799f, 0.2426111251115799f));
  q = ffma2(q, f, f2_pack(0.6932609677314758f, 0.6932609677314758f));
  q = ffma2(q, f, f2_pack(0.9999280571937561f, 0.9999280571937561f));
  float t0, t1;
  f2_unpack(t, t0, t1);
  q = fmul2(q, f2_pack(__int_as_float(__float_as_int(t0) << 23),
                       __int_as_float(__float_as_int(t1) << 23)));
  f2_unpack(q, r0, r1);
}

// ---------------------------------------------------------------------------
// The kernel
// ---------------------------------------------------------------------------
template <int D>
struct Cfg {
  static constexpr int kTileBytes = kRows * D * 2;
  static constexpr int kStages = D == 128 ? 4 : 8;       // K and V tiles in the ring
  static constexpr int kQOff = 0;
  static constexpr int kKVOff = 2 * kTileBytes;
  static constexpr int kOutOff = kKVOff + kStages * kTileBytes;   // each warp's 32 x 64 outputs
  static constexpr int kOutWarp = 32 * 64 * 2;
  static constexpr int kBarOff = kOutOff + 8 * kOutWarp;
  // q, kv_full[], kv_empty[], s_full[2], p_full[2], o_full[2], drain, p_half[2],
  // q_empty, unit_full[2], unit_empty[2], v_raw
  static constexpr int kNumBars = 1 + 2 * kStages + 15;
  static constexpr int kPieceOff = kBarOff + (kNumBars * 8 + 15) / 16 * 16;
  static constexpr int kMiscOff = kPieceOff + 2 * sizeof(Piece);
  static constexpr int kSmemBytes = kMiscOff + 16 + 1024;   // + alignment slack
  static constexpr int kSlot = 2 * kRows * (D + 2);         // floats of a unit's part
  __device__ static constexpr uint32_t col_s(int t) { return 128u * t; }
  __device__ static constexpr uint32_t col_o(int t) { return 256u + D * t; }
};

// A wait on the way out: ends with the phase or after a short limit.
__device__ __forceinline__ void last_wait(uint32_t bar, uint32_t parity) {
  const unsigned long long t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer_ns() - t0 > 50ull * 1000ull * 1000ull) return;
}

template <int D, bool F16>
__global__ void __launch_bounds__(kThreads, 1)
    paged_tiles_kernel(const __grid_constant__ CUtensorMap tmQ,
                       const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const TileParams p) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t sQ = base + C::kQOff;
  const uint32_t sKV = base + C::kKVOff;
  const uint32_t bars = base + C::kBarOff;
  constexpr int kB0 = 1 + 2 * C::kStages;
  const uint32_t bar_q = bars;
  auto bar_kv_full = [&](int s) { return bars + 8u * (1 + s); };
  auto bar_kv_empty = [&](int s) { return bars + 8u * (1 + C::kStages + s); };
  auto bar_s_full = [&](int t) { return bars + 8u * (kB0 + t); };
  auto bar_p_full = [&](int t) { return bars + 8u * (kB0 + 2 + t); };
  auto bar_o_full = [&](int t) { return bars + 8u * (kB0 + 4 + t); };
  const uint32_t bar_drain = bars + 8u * (kB0 + 6);
  auto bar_p_half = [&](int t) { return bars + 8u * (kB0 + 7 + t); };   // keys 0-63 of P_t
  const uint32_t bar_q_empty = bars + 8u * (kB0 + 9);   // the unit's last S products are done
  auto bar_unit_full = [&](int s) { return bars + 8u * (kB0 + 10 + s); };
  auto bar_unit_empty = [&](int s) { return bars + 8u * (kB0 + 12 + s); };
  const uint32_t bar_v_raw = bars + 8u * (kB0 + 14);    // a V tile whose end is to be zeroed
  // Ring of two pieces; h = -1 ends the CTA's work.
  volatile Piece* ring = reinterpret_cast<volatile Piece*>(gbase + C::kPieceOff);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + C::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + C::kMiscOff + 4);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  grid_dependents_launch();
  if (threadIdx.x == 0) {
    mbar_init(bar_q, 1);
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(bar_kv_full(s), 1);
      mbar_init(bar_kv_empty(s), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar_s_full(t), 1);
      mbar_init(bar_p_full(t), kRows);
      mbar_init(bar_p_half(t), kRows);
      mbar_init(bar_o_full(t), 1);
      mbar_init(bar_unit_full(t), 1);
      mbar_init(bar_unit_empty(t), 1 + 1 + 8);
    }
    mbar_init(bar_drain, 1);
    mbar_init(bar_q_empty, 1);
    mbar_init(bar_v_raw, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  // Rows of the Q tiles that no load writes (128 - g * floor(128 / g)) stay zero.
  for (int i = threadIdx.x; i < 2 * C::kTileBytes / 16; i += kThreads)
    *reinterpret_cast<uint4*>(gbase + C::kQOff + i * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();               // the plan is complete

  int raws = 0;         // V tiles whose end was zeroed

  // Warp-uniform bounded wait: every lane waits, and the warp goes on only if
  // all saw the phase, so that giving up never splits a warp.
  auto wwait = [&](uint32_t bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.status));
  };

  // K (kv = 0) or V (1) tiles of the n key blocks from blk0, by one warp: one
  // lane per page.  Block i of the CTA goes to ring position 2 i + kv.
  auto load_keys = [&](const CUtensorMap* map, int kv, int b, int h, int kv_len, int blk0, int n,
                       int& blocks) {
    const uint64_t policy = l2_policy_evict_last();
    const int boxes = kKeys / p.box_rows;
    const int in_page = (1 << p.page_shift) - p.box_rows;      // mask of a box's row in its page
    const uint32_t box_bytes = static_cast<uint32_t>(p.box_rows) * 128u;
    const int32_t* trow = p.table + b * p.table_stride;
    // Page of this lane's box of block j; one outside the cache reads as zeros.
    auto page_for = [&](int j) {
      const int key = j * kKeys + lane * p.box_rows;
      if (lane >= boxes || key >= kv_len) return p.pages;
      const int pg = page_at(trow, key, p.page_shift, p.max_pages, p.pages);
      if (pg < 0) atomicMax(p.status, kDevBadPage);
      return pg < 0 ? p.pages : pg;
    };
    int page = page_for(blk0);
    for (int j = blk0; j < blk0 + n; ++j, ++blocks) {
      const int page_next = j + 1 < blk0 + n ? page_for(j + 1) : 0;
      const int keys = min(kKeys, kv_len - j * kKeys);          // > 0
      const int used = (keys + p.box_rows - 1) / p.box_rows;
      const int pos = 2 * blocks + kv;
      const int s = pos % C::kStages;
      const uint32_t phase = (pos / C::kStages) & 1;
      if (!wwait(bar_kv_empty(s), phase ^ 1u)) return false;
      const uint32_t dst = sKV + s * C::kTileBytes;
      // A V tile that ends inside is handed on after its end is zeroed.
      const bool cut = kv == 1 && keys < kKeys;
      const uint32_t bar = cut ? bar_v_raw : bar_kv_full(s);
      if (lane == 0) mbar_arrive_expect_tx(bar, used * box_bytes * (D / 64));
      __syncwarp();
      if (lane < used) {
#pragma unroll
        for (int dk = 0; dk < D / 64; ++dk)
          tma_load_4d(dst + dk * 16384 + lane * box_bytes, map, bar, dk * 64,
                      (j * kKeys) & in_page, h, page, policy);
      }
      if (cut) {
        if (!wwait(bar_v_raw, raws & 1)) return false;
        ++raws;
        uint8_t* v = gbase + C::kKVOff + s * C::kTileBytes;
        for (int i = keys * 8 + lane; i < kKeys * 8; i += 32)
#pragma unroll
          for (int dk = 0; dk < D / 64; ++dk)
            *reinterpret_cast<uint4*>(v + dk * 16384 + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_kv_full(s));
      }
      page = page_next;
    }
    return true;
  };
  // On the way out: waits for a loader's last copies.
  auto land = [&](int kv, int blocks) {
    if (kv == 1) last_wait(bar_v_raw, raws & 1);
    for (int i = max(0, blocks - C::kStages / 2); i < blocks; ++i)
      last_wait(bar_kv_full((2 * i + kv) % C::kStages), ((2 * i + kv) / C::kStages) & 1);
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsCtrl) : "memory");
    if (warp == 8) {
      // =================== loads of Q and K ===================
      // (all loaded at once, whichever of them are used)
      const int4 plan0 = reinterpret_cast<const int4*>(p.plan)[0];
      const int4 plan1 = reinterpret_cast<const int4*>(p.plan)[1];
      const int first = p.first[blockIdx.x], behind = p.first[blockIdx.x + 1];
      static_assert(kSplit == 0 && kUnits == 3 && kPieces == 4 && kLongest == 5, "header words");
      const bool split = plan0.x != 0;
      const int pieces = split ? 0 : plan1.x, longest = plan1.y;
      int64_t next = split ? first : static_cast<int>(blockIdx.x);
      const int64_t stop = split ? behind : static_cast<int64_t>(pieces) + plan0.w;
      auto take_next = [&] {
        if (split) return next + 1;
        int got = 0;
        if (lane == 0) got = atomicAdd(p.plan + kNext, 1);
        return static_cast<int64_t>(gridDim.x) + __shfl_sync(0xffffffffu, got, 0);
      };
      const uint64_t pol_q = l2_policy_evict_first();
      int blocks = 0;       // K tiles issued, over all pieces
      int uc = 0;           // pieces with keys
      for (int take = 0;; ++take) {
        const int us = take & 1;
        if (take >= 2 && !wwait(bar_unit_empty(us), ((take >> 1) - 1) & 1)) break;
        Piece x;
        x.h = -1;
        for (; next < stop; next = take_next()) {
          x = split || next < pieces ? p.pieces[next] : whole_unit(p, next - pieces);
          // (a unit whose parts are pieces is not taken whole)
          if (split || next < pieces || max(x.nt[0], x.nt[1]) <= longest) break;
          x.h = -1;
        }
        if (lane == 0) {
          volatile Piece* d = ring + us;
          d->b = x.b;
          d->h = x.h;
          d->tok0 = x.tok0;
          d->q_begin = x.q_begin;
          d->q_len = x.q_len;
          d->kv_len = x.kv_len;
          d->blk0 = x.blk0;
          d->nt[0] = x.nt[0];
          d->nt[1] = x.nt[1];
          d->slot = x.slot;
          d->place0 = x.place0;
          mbar_arrive(bar_unit_full(us));
        }
        if (x.h < 0) break;
        const int n = max(x.nt[0], x.nt[1]);
        if (n > 0) {
          // The Q tiles are free once the last piece's S products are done.
          if (uc > 0 && !wwait(bar_q_empty, (uc - 1) & 1)) break;
          if (lane == 0) {
            const uint32_t bytes = static_cast<uint32_t>(p.tq) * p.g * 128u * (D / 64);
            mbar_arrive_expect_tx(bar_q, bytes * ((x.nt[0] > 0 ? 1 : 0) + (x.nt[1] > 0 ? 1 : 0)));
#pragma unroll
            for (int t = 0; t < 2; ++t)
              if (x.nt[t] > 0)
#pragma unroll
                for (int dk = 0; dk < D / 64; ++dk)
                  tma_load_4d(sQ + t * C::kTileBytes + dk * 16384, &tmQ, bar_q, dk * 64, 0,
                              x.q_begin + x.tok0 + t * p.tq, x.h, pol_q);
          }
          ++uc;
          if (!load_keys(&tmK, 0, x.b, x.h, x.kv_len, x.blk0, n, blocks)) break;
        }
        next = take_next();
      }
      if (*abort_flag && lane == 0) {
        // Let the copies in flight land before the CTA exits.
        if (uc > 0) last_wait(bar_q, (uc - 1) & 1);
        land(0, blocks);
      }
      __syncwarp();
    } else if (warp == 10) {
      // =================== loads of V ===================
      int blocks = 0;
      for (int uc = 0;; ++uc) {
        const int us = uc & 1;
        if (!wwait(bar_unit_full(us), (uc >> 1) & 1)) break;
        const int b = ring[us].b, h = ring[us].h, kv_len = ring[us].kv_len;
        const int blk0 = ring[us].blk0, n = max(ring[us].nt[0], ring[us].nt[1]);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_unit_empty(us));
        if (h < 0) break;
        if (n > 0 && !load_keys(&tmV, 1, b, h, kv_len, blk0, n, blocks)) break;
      }
      if (*abort_flag && lane == 0) land(1, blocks);
      __syncwarp();
    } else if (warp == 9) {
      // =================== MMA issuer ===================
      if (elect_one()) {
        constexpr uint32_t kIdQK = idesc_f32acc(kRows, kKeys, false, false, F16);
        constexpr uint32_t kIdPV = idesc_f32acc(kRows, D, false, true, F16);
        bool ok = true;
        int it = 0;              // K and V tiles taken, over all pieces
        int uq = 0;              // pieces with keys
        int pb[2] = {0, 0};      // key blocks of tile t in earlier pieces (P phases)
        for (int uc = 0; ok; ++uc) {
          const int us = uc & 1;
          if (!mbar_wait(bar_unit_full(us), (uc >> 1) & 1, abort_flag, p.status)) break;
          const int h = ring[us].h;
          const int nt[2] = {ring[us].nt[0], ring[us].nt[1]};
          mbar_arrive(bar_unit_empty(us));
          if (h < 0) break;
          const int n = max(nt[0], nt[1]);
          if (n == 0) continue;
          if (!mbar_wait(bar_q, uq & 1, abort_flag, p.status)) break;
          ++uq;
          tc_fence_after();
          int vslot = 0;
          for (int j = 0; ok && j <= n; ++j) {
            int kslot = 0;
            if (j < n) {
              kslot = it % C::kStages;
              if (!mbar_wait(bar_kv_full(kslot), (it / C::kStages) & 1, abort_flag, p.status)) {
                ok = false;
                break;
              }
              ++it;
              tc_fence_after();
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (j >= 1 && j - 1 < nt[t]) {
                // O_t += P_t(j-1) V_{j-1}: P from TMEM, V with D contiguous; the
                // first 64 keys go as soon as their half of P is stored.
                const uint32_t vbase = sKV + vslot * C::kTileBytes;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  const uint32_t bar = half == 0 ? bar_p_half(t) : bar_p_full(t);
                  if (!mbar_wait(bar, (pb[t] + j - 1) & 1, abort_flag, p.status)) {
                    ok = false;
                    break;
                  }
                  tc_fence_after();
#pragma unroll
                  for (int kk = half * 4; kk < half * 4 + 4; ++kk)
                    mma_ts(tmem + C::col_o(t), tmem + C::col_s(t) + kk * 8,
                           sdesc_sw128(vbase + kk * 2048, 16384, 1024), kIdPV,
                           (j - 1 > 0 || kk > 0) ? 1u : 0u);
                }
                if (!ok) break;
                if (j - 1 == nt[t] - 1) mma_commit(bar_o_full(t));
              }
              if (j < nt[t]) {
                // S_t = Q_t K_j^T, both with D contiguous.
                const uint32_t qbase = sQ + t * C::kTileBytes;
                const uint32_t kbase = sKV + kslot * C::kTileBytes;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                  const uint32_t off = (kk >> 2) * 16384 + (kk & 3) * 32;
                  mma_ss(tmem + C::col_s(t), sdesc_sw128(qbase + off, 16, 1024),
                         sdesc_sw128(kbase + off, 16, 1024), kIdQK, kk > 0 ? 1u : 0u);
                }
                mma_commit(bar_s_full(t));
              }
            }
            if (!ok) break;
            if (j >= 1) mma_commit(bar_kv_empty(vslot));
            if (j < n) {
              mma_commit(bar_kv_empty(kslot));
              if (j == n - 1) mma_commit(bar_q_empty);
              vslot = it % C::kStages;
              if (!mbar_wait(bar_kv_full(vslot), (it / C::kStages) & 1, abort_flag, p.status)) {
                ok = false;
                break;
              }
              ++it;
              tc_fence_after();
            }
          }
          pb[0] += nt[0];
          pb[1] += nt[1];
        }
        // Every issued MMA and its arrivals complete before teardown.
        mma_commit(bar_drain);
        last_wait(bar_drain, 0);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax) : "memory");
    // =================== softmax, rescaling, output ===================
    const int t = warp >> 2;
    const int wq = warp & 3;
    const int row = wq * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t tS = tmem + lane_off + C::col_s(t);
    const uint32_t tO = tmem + lane_off + C::col_o(t);
    const float sl2 = p.scale_log2;
    const uint64_t sl2x2 = f2_pack(sl2, sl2);
    const int row_tok = row / p.g;
    bool ok = true;
    int sb = 0;   // key blocks of this tile in earlier pieces (S phases)
    int ou = 0;   // earlier pieces in which this tile had keys (O phases)
    for (int uc = 0; ok; ++uc) {
      const int us = uc & 1;
      if (!wwait(bar_unit_full(us), (uc >> 1) & 1)) break;
      if (ring[us].h < 0) break;
      const int kv_len = ring[us].kv_len, blk0 = ring[us].blk0, nt = ring[us].nt[t];
      // Keys [0, lim) are seen by this row; no row of the tile sees fewer than lim0.
      int lim = kv_len, lim0 = kv_len;
      bool any_live;
      {
        const int tok_t = ring[us].tok0 + t * p.tq, q_len = ring[us].q_len;
        const bool live = row_tok < p.tq && tok_t + row_tok < q_len;
        if (p.causal && tok_t < q_len) lim0 = ring[us].place0 + tok_t + 1;
        if (p.causal && live) lim = min(kv_len, lim0 + row_tok);
        any_live = __any_sync(0xffffffffu, live);
      }
      float m_ref = -INFINITY;   // reference maximum (scaled, log2 domain)
      float l = 0.f;             // sum of exp2(s * sl2 - m_ref)
      for (int j = 0; j < nt; ++j) {
        if (!wwait(bar_s_full(t), (sb + j) & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (!any_live) {         // rows of no token: whatever their P holds stays in their O
          mbar_arrive(bar_p_half(t));
          mbar_arrive(bar_p_full(t));
          continue;
        }
        uint32_t sr[128];
        tmem_ld128_wait(tS, sr);
        const int k0 = (blk0 + j) * kKeys;
        if (k0 + kKeys > lim0 || k0 + kKeys > kv_len) {
#pragma unroll
          for (int c = 0; c < kKeys; ++c)
            if (k0 + c >= lim) sr[c] = __float_as_uint(-INFINITY);
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < kKeys; c += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mx4[i] = max3(mx4[i], __uint_as_float(sr[c + 2 * i]), __uint_as_float(sr[c + 2 * i + 1]));
        const float m_blk = max3(max3(mx4[0], mx4[1], mx4[2]), mx4[3], -INFINITY) * sl2;
        // The reference is raised only when a row outgrows it by 2^8, so that
        // O is rarely rescaled; O / l is exact for any reference.
        const bool need = !(m_blk <= m_ref + 8.f);
        if (__any_sync(0xffffffffu, need)) {
          const float m_use = need ? m_blk : m_ref;
          const float alpha = m_use == -INFINITY   ? 1.f
                              : m_ref == -INFINITY ? 0.f
                                                   : ex2_approx(m_ref - m_use);
          if (j > 0) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32_wait(tO + c * 32, o);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st32(tO + c * 32, o);
            }
          }
          l *= alpha;
          m_ref = m_use;
        }
        const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref;
        const uint64_t negm2 = f2_pack(neg_m, neg_m);
        uint64_t rs2[2] = {0ull, 0ull};
        uint32_t pk[2][32];
        auto exp_half = [&](int half) {
#pragma unroll
          for (int cc = 0; cc < 32; ++cc) {
            const int c = half * 32 + cc;
            float x0, x1, p0, p1;
            f2_unpack(ffma2(f2_pack(__uint_as_float(sr[2 * c]), __uint_as_float(sr[2 * c + 1])),
                            sl2x2, negm2),
                      x0, x1);
            if (c % 4 == 3) {
              exp2_pair(x0, x1, p0, p1);
            } else {
              p0 = ex2_approx(x0);
              p1 = ex2_approx(x1);
            }
            rs2[c & 1] = fadd2(rs2[c & 1], f2_pack(p0, p1));
            pk[half][cc] = pack_16x2<F16>(p0, p1);
          }
        };
        exp_half(0);
        tmem_st32(tS, pk[0]);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar_p_half(t));
        exp_half(1);
        float a0, a1, b0, b1;
        f2_unpack(rs2[0], a0, a1);
        f2_unpack(rs2[1], b0, b1);
        l += (a0 + a1) + (b0 + b1);
        tmem_st32(tS + 32, pk[1]);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar_p_full(t));
      }
      if (!ok) break;
      if (nt > 0) {
        if (!wwait(bar_o_full(t), ou & 1)) break;
        tc_fence_after();
        ++ou;
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int h = ring[us].h, q_begin = ring[us].q_begin, slot = ring[us].slot;
      const int tok = ring[us].tok0 + t * p.tq + row_tok;
      const bool live = row_tok < p.tq && tok < ring[us].q_len;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_unit_empty(us));
      if (slot < 0) {
        // 32 rows x 64 outputs at a time through shared memory (16-byte chunks
        // swizzled by the row), so that a store covers 128 bytes of each of 4
        // rows instead of 16 of 32.
        uint8_t* stage = gbase + C::kOutOff + warp * C::kOutWarp;
        const int64_t off = live ? static_cast<int64_t>(q_begin + tok) * p.o_st +
                                       static_cast<int64_t>(h * p.g + row - row_tok * p.g) * p.o_sh
                                 : -1;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          uint32_t o[64];
          if (nt > 0) {
            tmem_ld64_wait(tO + c * 64, o);
          } else {
#pragma unroll
            for (int e = 0; e < 64; ++e) o[e] = 0u;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = pack_16x2<F16>(__uint_as_float(o[e * 8 + 2 * i]) * inv,
                                    __uint_as_float(o[e * 8 + 2 * i + 1]) * inv);
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((e ^ (lane & 7)) * 16)) =
                make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
          const int d = c * 64 + (lane & 7) * 8;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + lane / 8;
            const int64_t to = __shfl_sync(0xffffffffu, off, r);
            const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 +
                                                            (((lane & 7) ^ (r & 7)) * 16));
            if (to >= 0 && d < p.D)
              *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.o) + to + d) = v;
          }
          __syncwarp();
        }
      } else {
        // Four channels of 32 rows side by side: 512 bytes per store.
        float* part = p.part + static_cast<int64_t>(slot) * C::kSlot;
        if (nt > 0) {
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32_wait(tO + c * 32, o);
            uint4* dst = reinterpret_cast<uint4*>(part) + (t * (D / 4) + c * 8) * kRows + row;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (live)
                dst[e * kRows] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        }
        if (live) {
          part[2 * kRows * D + t * kRows + row] = m_ref;
          part[2 * kRows * D + 2 * kRows + t * kRows + row] = l;
        }
      }
      sb += nt;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Adds up the parts of a unit: a CTA takes 32 rows (a lane each), a warp D / 8
// channels of them.
// Bound by HBM: each part is read once.
constexpr int kJoinWarps = 8;
constexpr int kJoinGroups = 2 * kRows / 32;             // groups of 32 rows of a unit
template <int D, bool F16>
__global__ void __launch_bounds__(32 * kJoinWarps)
    paged_tiles_join(const TileParams p) {
  using C = Cfg<D>;
  constexpr int E = D / 4 / kJoinWarps;               // groups of four channels of a warp
  constexpr int kRowBytes = D * 2 + 16;
  __shared__ __align__(16) uint8_t s_out[32 * kRowBytes];
  __shared__ int64_t s_off[32];
  grid_dependency_wait();
  grid_dependents_launch();
  const int items = p.plan[kJoins] * kJoinGroups;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int4 j0 = reinterpret_cast<const int4*>(p.join + item / kJoinGroups)[0];
    const int4 j1 = reinterpret_cast<const int4*>(p.join + item / kJoinGroups)[1];
    const int slot0 = j0.x, parts = j0.y, tok0 = j0.z, q_begin = j0.w, q_len = j1.x, h = j1.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = item % kJoinGroups / (kRows / 32);
    const int row = item % (kRows / 32) * 32 + lane;            // of the tile
    const int row_tok = row / p.g;
    const int tok = tok0 + t * p.tq + row_tok;
    const bool live = row_tok < p.tq && tok < q_len;
    if (!__any_sync(0xffffffffu, live)) continue;               // (the same in every warp)
    const float* part = p.part + static_cast<int64_t>(slot0) * C::kSlot;
    const int at_m = 2 * kRows * D + t * kRows + row, at_l = at_m + 2 * kRows;
    const int at_o = (t * (D / 4) + warp * E) * kRows + row;
    float top = -INFINITY, sum = 0.f;
    float4 acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    // kAhead parts at a time, all of their loads in flight together.
    constexpr int kAhead = 4;
    for (int i0 = 0; live && i0 < parts; i0 += kAhead) {
      float m[kAhead], l[kAhead];
      float4 o[kAhead][E];
      float now = top;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const bool in = i0 + k < parts;
        const float* s = part + static_cast<int64_t>(in ? i0 + k : i0) * C::kSlot;
        m[k] = in ? s[at_m] : -INFINITY;
        l[k] = in ? s[at_l] : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[k][e] = reinterpret_cast<const float4*>(s)[at_o + e * kRows];
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) now = fmaxf(now, m[k]);
      const float keep = top == -INFINITY ? 0.f : ex2_approx(top - now);
      sum *= keep;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        acc[e].x *= keep;
        acc[e].y *= keep;
        acc[e].z *= keep;
        acc[e].w *= keep;
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (m[k] == -INFINITY) {          // saw none of these keys: O was not written
          sum += l[k];
          continue;
        }
        const float al = ex2_approx(m[k] - now);
        sum += l[k] * al;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          acc[e].x += o[k][e].x * al;
          acc[e].y += o[k][e].y * al;
          acc[e].z += o[k][e].z * al;
          acc[e].w += o[k][e].w * al;
        }
      }
      top = now;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int e = 0; e < E; ++e)
      *reinterpret_cast<uint2*>(s_out + lane * kRowBytes + (warp * E + e) * 8) =
          make_uint2(pack_16x2<F16>(acc[e].x * inv, acc[e].y * inv),
                     pack_16x2<F16>(acc[e].z * inv, acc[e].w * inv));
    if (warp == 0)
      s_off[lane] = live ? static_cast<int64_t>(q_begin + tok) * p.o_st +
                               static_cast<int64_t>(h * p.g + row - row_tok * p.g) * p.o_sh
                         : -1;
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * (D / 8); i += 32 * kJoinWarps) {
      const int r = i / (D / 8), d = (i - r * (D / 8)) * 8;
      if (s_off[r] >= 0 && d < p.D)
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.o) + s_off[r] + d) =
            *reinterpret_cast<const uint4*>(s_out + r * kRowBytes + d * 2);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int tile_tokens(const fa_paged_attn_args* a) {
  return static_cast<int>(kRows / (a->Hq / a->Hkv));
}

PlanOffsets plan_offsets(const fa_paged_attn_args* a, int sms) {
  PlanOffsets o;
  o.prefix = up128(kHeader * 4);
  o.first = o.prefix + up128((a->B + 1) * 4);
  o.join = o.first + up128((sms + 1) * 4);
  o.pieces = o.join + up128(sms * static_cast<int64_t>(sizeof(JoinUnit)));
  o.parts = o.pieces + up128((kUnitsPerSm + 1) * sms * static_cast<int64_t>(sizeof(Piece)));
  const int d = a->D <= 64 ? 64 : 128;
  o.bytes = o.parts + 2ll * sms * 2 * kRows * (d + 2) * 4;   // a CTA ends and begins a part
  return o;
}

// 4-D tensor map of 16-bit elements, innermost dimension first, boxes of 64
// channels (128-byte swizzle).  A dimension of one entry gets a legal stride.
int make_map(CUtensorMap* map, const void* ptr, const int64_t (&dims)[4],
             const int64_t (&strides)[3], const uint32_t (&box)[3], bool f16) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (enc == nullptr) return FA_ERR_DRIVER;
  cuuint64_t d[4], s[3];
  cuuint32_t b[4] = {64, box[0], box[1], box[2]}, one[4] = {1, 1, 1, 1};
  for (int i = 0; i < 4; ++i) d[i] = static_cast<cuuint64_t>(dims[i]);
  for (int i = 0; i < 3; ++i) s[i] = dims[i + 1] > 1 ? static_cast<cuuint64_t>(strides[i]) * 2 : 256;
  const CUresult r =
      enc(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
          const_cast<void*>(ptr), d, s, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FA_OK : FA_ERR_TMA;
}

template <int D, bool F16>
int launch_tiles(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                 const TileParams& p, cudaStream_t stream) {
  using C = Cfg<D>;
  static KernelPrep prep;
  int dev = 0;
  int rc = prepare_kernel(prep, reinterpret_cast<const void*>(paged_tiles_kernel<D, F16>),
                          C::kSmemBytes, &dev);
  if (rc != FA_OK) return rc;
  rc = launch_after(paged_plan_kernel, dim3(1), kPlanThreads, 0, 1, stream, p);
  if (rc != FA_OK) return rc;
  rc = launch_after(paged_tiles_kernel<D, F16>, dim3(p.ctas), kThreads, C::kSmemBytes, 1, stream, mq,
                    mk, mv, p);
  if (rc != FA_OK) return rc;
  return launch_after(paged_tiles_join<D, F16>, dim3(2 * p.ctas),
                      32 * kJoinWarps, 0, 1, stream, p);
}

}  // namespace

int64_t paged_tiles_bytes(const fa_paged_attn_args* a, int sms) {
  return plan_offsets(a, sms).bytes;
}

int launch_paged_tiles(const fa_paged_attn_args* a, const PagedParams& q, void* workspace,
                       cudaStream_t stream) {
  TileParams p;
  static_cast<PagedParams&>(p) = q;
  p.tq = tile_tokens(a);
  p.box_rows = a->page_size < kKeys ? static_cast<int>(a->page_size) : kKeys;
  const PlanOffsets o = plan_offsets(a, p.ctas);
  char* ws = static_cast<char*>(workspace);
  p.plan = reinterpret_cast<int*>(ws);
  p.prefix = reinterpret_cast<int*>(ws + o.prefix);
  p.first = reinterpret_cast<int*>(ws + o.first);
  p.join = reinterpret_cast<JoinUnit*>(ws + o.join);
  p.pieces = reinterpret_cast<Piece*>(ws + o.pieces);
  p.part = reinterpret_cast<float*>(ws + o.parts);
  p.min_cells = 4;
  p.split_units = kUnitsPerSm * p.ctas;
  if (p.split_units > kPlanThreads) p.split_units = kPlanThreads;
  if (p.ctas > kMaxSplitCtas) p.split_units = 0;
  CUtensorMap mq, mk, mv;
  const bool f16 = a->dtype == FA_F16;
  const int64_t g = a->Hq / a->Hkv;
  int rc = make_map(&mq, a->q, {a->D, g, a->T, a->Hkv},
                    {a->q_strides[1], a->q_strides[0], a->q_strides[1] * g},
                    {static_cast<uint32_t>(g), static_cast<uint32_t>(p.tq), 1}, f16);
  if (rc != FA_OK) return rc;
  const uint32_t rows = static_cast<uint32_t>(p.box_rows);
  const int64_t dims[4] = {a->D, a->page_size, a->Hkv, a->pages};
  rc = make_map(&mk, a->k_cache, dims,
                {a->k_cache_strides[1], a->k_cache_strides[2], a->k_cache_strides[0]},
                {rows, 1, 1}, f16);
  if (rc != FA_OK) return rc;
  rc = make_map(&mv, a->v_cache, dims,
                {a->v_cache_strides[1], a->v_cache_strides[2], a->v_cache_strides[0]},
                {rows, 1, 1}, f16);
  if (rc != FA_OK) return rc;
  if (a->D <= 64)
    return f16 ? launch_tiles<64, true>(mq, mk, mv, p, stream)
               : launch_tiles<64, false>(mq, mk, mv, p, stream);
  return f16 ? launch_tiles<128, true>(mq, mk, mv, p, stream)
             : launch_tiles<128, false>(mq, mk, mv, p, stream);
}

}  // namespace fa
