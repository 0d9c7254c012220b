// Shared declarations of the attention over a shared prefix and per-sequence
// caches (attn_cached.cu, attn_prefix_tc.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "longctx.h"

namespace inf {

// Query rows are numbered r = (b * n_tokens + t) * n_heads + h.  A CTA leaves, for
// each of its rows, one partial result over its keys: the largest logit (or a reference
// near it, below) and the sum and weighted V sum of exp2(logit - that); logits are in
// units of log2.
//
// The prefix is cut into p_splits equal splits; row r's partial of split s is entry
// r * p_splits + s.  The own parts are cut evenly whatever lens are: keys are counted
// in blocks of AC_BLOCK, the sequences' blocks stand in one line, and group c of
// o_groups takes `share` blocks of it from c * share on, with one CTA for each unit:
// a KV head and a row tile of o_rows rows.  (The CTAs of a group walk the same keys
// side by side, so that the heads' parts of a cache row are read together.)  Along
// the line either the group or the sequence steps, so group c's partials of sequence
// b are slot c + b: units * o_rows entries from own_base on.  head holds share and
// the blocks before each sequence.
struct AcParams {
  const void* q;
  const void *pk, *pv;           // shared prefix [prefix_len][nkv][hd]
  const void *kc, *vc;           // own slices [max_len][nkv][hd], seq_stride apart
  const int* lens;
  void* out;
  float* scores;
  long long q_stride, out_stride, seq_stride, score_stride;   // elements
  int batch, n_tok, nh, nkv, group, prefix_len, max_len;
  FastDiv by_seq, by_group;      // a sequence's rows of one KV head, n_tok * group; group
  FastDiv by_groups;             // o_groups
  float scale_log2;              // scale * log2(e)
  int p_splits, p_split_len;     // split s: keys [s * len, (s + 1) * len)
  int o_rows, o_tiles, o_groups;
  long long own_base;
  float* part_o;                 // [entry][hd]
  float2* part_ml;               // [entry] (largest logit, sum)
  int* head;                     // [1 + batch]
  float* logits;                 // [row][logit_stride] own logits (only with scores)
  long long logit_stride;
};

// What a row's logits are taken relative to when the largest is `top`: that less `exp`,
// so that the largest P is 2^exp.  From 2^22 on, where fp32 has no room for the
// difference, top itself.
constexpr float AC_FAR = 4194304.f;
template <int exp>
__device__ __forceinline__ float ac_ref(float top) {
  return exp && fabsf(top) < AC_FAR ? top - (float)exp : top;
}

constexpr int AC_BLOCK = 64;
constexpr float AC_LOG2E = 1.4426950408889634f;

// 16 bytes to shared memory, zeros where not valid (src is then not read)
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// the prefix part on tcgen05 (attn_prefix_tc.cu): query rows per CTA, CTAs per SM
int ap_rows();
int ap_ctas_per_sm(int hd);
// give_up: every wait that the work depends on runs out at once (a test of that path)
int launch_attn_prefix_tc(int type, int hd, const AcParams& p, int row_tiles, bool give_up, cudaStream_t st);

}  // namespace inf
