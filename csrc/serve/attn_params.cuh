// Arguments and pieces of the decoding attention, shared by its kernels.
#pragma once
#include "f32x2.cuh"

namespace hb {

struct KvView {
  const uint8_t *k, *v;
  const int8_t *ke, *ve;
  long long kb, ks, kn, vb, vs, vn;          // bytes
  long long keb, kes, ken, veb, ves, ven;    // elements
};
struct AttnParams {
  const __nv_bfloat16* q;
  long long qb, qs, qh;
  KvView own, pre;
  const int *lengths, *counts;
  int B, S, Nq, N, G, C, P, W;
  int pre_lo;                 // first prefix key that any query can see
  float sl2;                  // scale * log2(e)
  // prefix pieces on mma.sync: CTAs, key splits, row tiles
  int n_pre, n_split, pre_rt;
  // prefix pieces on tcgen05: CTAs, tiles per CTA, tiles and row tiles per KV head, rows of a row tile
  int tc_ctas, tc_per, tc_tiles, tc_rt, tc_rows;
  int n_suf, own_rt;          // own-key CTAs per (KV head, row tile); row tiles of a sequence
  float *own_o, *own_ml, *pre_o, *pre_ml;
  int* tile_start;            // [B + 1]
  __nv_bfloat16* out;         // [B, S, Nq, H] contiguous
  int* status;
  unsigned long long budget_ns;
};

HB_DEVICE float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Programmatic launch: let the next kernel of the stream start / wait for the
// previous one's memory.
HB_DEVICE void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
HB_DEVICE void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

HB_DEVICE int len_of(const AttnParams& p, int b, bool report) {
  const int x = p.lengths[b], y = min(max(x, 0), p.C);
  if (report && x != y) set_error(p.status, kErrBounds);
  return y;
}
HB_DEVICE int count_of(const AttnParams& p, int b, int len, bool report) {
  if (!p.counts) return min(p.S, len);
  const int x = p.counts[b], y = min(max(x, 0), min(p.S, len));
  if (report && x != y) set_error(p.status, kErrBounds);
  return y;
}

// Prefix pieces of the rows of all sequences on tcgen05; head dim 64 or 128,
// bf16 keys and values (k, v: [P, N, H] with row and head strides in bytes).
void prefix_tc_launch(const AttnParams& p, int H, const void* k, const void* v, long long ks, long long kn, long long vs,
                      long long vn);

}  // namespace hb
