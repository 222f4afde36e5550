// What the row and tile kernels of the paged attention share.
#pragma once

#include "fa_internal.h"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace fa {

// Row kernel: the unit (rows of one head) that a CTA begins and others end.
struct OpenUnit {
  int parts;                            // 0: there is none
  int h, row0, rows, begin;             // head, rows of the sequence, its first token
  int pad[3];
};

struct PagedParams {
  const void* q;
  void* o;
  const void* kc;
  const void* vc;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;
  int64_t q_st, q_sh, o_st, o_sh;       // elements: token, head
  int64_t kc_p, kc_r, kc_h;             // page, row, head
  int64_t vc_p, vc_r, vc_h;
  int64_t table_stride;
  int T, B, Hkv, g, D;
  int pages, page_shift, max_pages;
  int causal;
  float scale_log2;
  int* status;
  float* part;                          // partial results of split units
  OpenUnit* open;                       // row kernel: one of each CTA, for the join
  int ctas;                             // ranges the key blocks are cut into
  int min_blocks;                       // least key blocks of a range
  int team;                             // row kernel: heads that stream side by side
  int tile_ctas;                        // row kernel, whole units: CTAs over a head's row tiles
  int cluster_shift;                    // and CTAs (1 << this) that share a unit's keys
};

// A sequence's new tokens and the keys that its table holds.
struct SeqWork {
  int begin, q_len, kv_len;
  int place0;            // the first new token's place: negative before the start, behind the
};                       // held keys where the length goes beyond the table

__device__ __forceinline__ SeqWork seq_work(const PagedParams& p, int b) {
  SeqWork w;
  const SeqRows r = seq_rows(p.cu, b, p.T);
  w.begin = r.begin;
  w.q_len = r.end - r.begin;
  const int len = p.lens[b];
  w.kv_len = held_len(len, p.page_shift, p.max_pages);
  if (len > w.kv_len && len > 0) atomicMax(p.status, kDevBadPage);
  w.place0 = max(len, 0) - w.q_len;
  return w;
}

// Keys [0, limit) that token i of the sequence sees.
__device__ __forceinline__ int seen_keys(const PagedParams& p, const SeqWork& w, int i) {
  return p.causal ? min(w.kv_len, max(0, w.place0 + i + 1)) : w.kv_len;
}

// The tile kernel: bytes of its workspace, and its launches (p.ctas = SMs).
int64_t paged_tiles_bytes(const fa_paged_attn_args* a, int sms);
int launch_paged_tiles(const fa_paged_attn_args* a, const PagedParams& p, void* workspace,
                       cudaStream_t stream);

}  // namespace fa
