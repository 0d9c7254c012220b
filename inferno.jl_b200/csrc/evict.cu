// Eviction of cache rows by gathered attention weight (inferno_cache_evict).
//
// Kernel 1, one CTA per (sequence, KV head): ranks the rows and decides which
// stay.  The rank key is the score as an order-preserving 32-bit integer, in two
// classes (rows kept always come first), and the budget-th largest key is found
// by a radix select of four 8-bit digits; ties at that key go to the lowest rows.
// One pass in row order then numbers the holes (evicted rows before the budget)
// and the kept rows behind it; the i-th of these goes into the i-th hole, so the
// two lists have equal lengths and no row is both read and written.  Scores and
// positions are placed here.
// Kernel 2 moves the K and V rows by the two lists.
#include <algorithm>
#include "internal.h"
#include "common.cuh"
#include "longctx.h"
#include "../../include/inferno_b200.h"

namespace inf {

constexpr int EV_THREADS = 1024;
constexpr int EV_MOVE_THREADS = 256;

struct EvictParams {
  uint8_t *kc, *vc;
  long long seq_bytes, row_bytes;     // bytes between slices; between rows of one KV head
  int head_bytes;
  const float* scores;
  const int* pos;
  const int *lens, *next_pos;
  float* scores_out;
  int *pos_out, *lens_out;
  long long stride;                   // entries between (sequence, KV head) rows of scores / pos
  int batch, nkv, max_len, budget, n_sink, n_recent, max_moves;
  int* counts;                        // [batch * nkv] rows to move
  int* lists;                         // [batch * nkv][2][max_moves]: holes, sources
};

// larger is kept first; NaN below everything; -0 equal to 0
__device__ __forceinline__ uint32_t ev_key(float s) { return s != s ? 0u : float_ordered(s + 0.0f); }

__device__ __forceinline__ bool ev_always(const EvictParams& p, int pos, int recent_from) {
  return pos < p.n_sink || pos >= recent_from;
}

// exclusive sums of v over the CTA in thread order; total in *sum
__device__ __forceinline__ int2 ev_scan(int2 v, int2* warp_sums, int2* sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int2 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, x.x, o), b = __shfl_up_sync(0xffffffffu, x.y, o);
    if (lane >= o) x.x += a, x.y += b;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int2 before = make_int2(0, 0), all = make_int2(0, 0);
  for (int w = 0; w < EV_THREADS / 32; ++w) {
    const int2 s = warp_sums[w];
    if (w < warp) before.x += s.x, before.y += s.y;
    all.x += s.x, all.y += s.y;
  }
  *sum = all;
  return make_int2(before.x + x.x - v.x, before.y + x.y - v.y);
}

__global__ void __launch_bounds__(EV_THREADS) evict_select_kernel(const EvictParams p) {
  const int bh = blockIdx.x, b = bh / p.nkv, t = threadIdx.x;
  const int len = max(0, min(p.lens[b], p.max_len));
  const float* sc = p.scores + bh * p.stride;
  const int* ps = p.pos + bh * p.stride;
  float* so = p.scores_out + bh * p.stride;
  int* po = p.pos_out + bh * p.stride;
  if (len <= p.budget) {
    if (so != sc)
      for (int j = t; j < len; j += EV_THREADS) so[j] = sc[j];
    if (po != ps)
      for (int j = t; j < len; j += EV_THREADS) po[j] = ps[j];
    if (t == 0) p.counts[bh] = 0;
    return;
  }
  __shared__ int hist[256];
  __shared__ int2 warp_sums[EV_THREADS / 32];
  __shared__ int s_always, s_digit, s_need;
  const long long rf = (long long)p.next_pos[b] - p.n_recent;
  const int recent_from = (int)max(-2147483648ll, rf);
  if (t == 0) s_always = 0;
  __syncthreads();
  int n = 0;
  for (int j = t; j < len; j += EV_THREADS) n += ev_always(p, ps[j], recent_from);
  atomicAdd(&s_always, n);
  __syncthreads();
  // the class the border lies in: the rows kept always when there are more of
  // them than the budget, else the others
  const bool among_always = s_always > p.budget;
  int need = among_always ? p.budget : p.budget - s_always;
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (t < 256) hist[t] = 0;
    __syncthreads();
    for (int j = t; j < len; j += EV_THREADS) {
      const uint32_t k = ev_key(sc[j]);
      if (ev_always(p, ps[j], recent_from) == among_always && (shift == 24 || (k >> (shift + 8)) == prefix))
        atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (t == 0) {      // the digit whose bin the need-th largest key falls into
      int left = need, d = 255;
      while (d > 0 && hist[d] < left) left -= hist[d--];
      s_digit = d;
      s_need = left;
    }
    __syncthreads();
    prefix = (prefix << 8) | s_digit;
    need = s_need;
  }
  // kept: class above the border, or key > prefix, or one of the first `need`
  // rows with key == prefix
  int* holes = p.lists + (long long)bh * 2 * p.max_moves;
  int* from = holes + p.max_moves;
  int ties = 0, nh = 0, nf = 0;
  for (int j0 = 0; j0 < len; j0 += EV_THREADS) {
    const int j = j0 + t;
    bool keep = false, tie = false;
    float s = 0.f;
    int po_j = 0;
    if (j < len) {
      s = sc[j];
      po_j = ps[j];
      const uint32_t k = ev_key(s);
      const bool al = ev_always(p, po_j, recent_from);
      if (al != among_always) {
        keep = al;
      } else {
        keep = k > prefix;
        tie = k == prefix;
      }
    }
    int2 sum;
    const int2 tr = ev_scan(make_int2(tie, 0), warp_sums, &sum);
    if (tie) keep = ties + tr.x < need;
    ties += sum.x;
    const bool hole = j < p.budget && j < len && !keep, src = j >= p.budget && keep;
    const int2 r = ev_scan(make_int2(hole, src), warp_sums, &sum);
    if (hole) holes[nh + r.x] = j;
    if (j < p.budget && keep) so[j] = s, po[j] = po_j;
    nh += sum.x;
    __syncthreads();                 // this chunk's holes are listed
    if (src) {
      const int to = holes[nf + r.y];
      from[nf + r.y] = j;
      so[to] = s;
      po[to] = po_j;
    }
    nf += sum.y;
  }
  if (t == 0) p.counts[bh] = nf;
}

__global__ void __launch_bounds__(EV_MOVE_THREADS) evict_move_kernel(const EvictParams p, int rows_per_block) {
  const int bh = blockIdx.y, b = bh / p.nkv, h = bh - b * p.nkv;
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0)
    p.lens_out[b] = min(max(0, min(p.lens[b], p.max_len)), p.budget);
  const int n = p.counts[bh];
  const int r0 = blockIdx.x * rows_per_block, r1 = min(n, r0 + rows_per_block);
  if (r0 >= r1) return;
  const int* holes = p.lists + (long long)bh * 2 * p.max_moves;
  const int* from = holes + p.max_moves;
  const int vecs = p.head_bytes / 16;
  uint8_t* base[2] = {p.kc + b * p.seq_bytes + (long long)h * p.head_bytes,
                      p.vc + b * p.seq_bytes + (long long)h * p.head_bytes};
  for (int i = threadIdx.x; i < (r1 - r0) * 2 * vecs; i += EV_MOVE_THREADS) {
    const int row = i / (2 * vecs), c = i - row * 2 * vecs, kv = c >= vecs;
    const long long off = (long long)(kv ? c - vecs : c) * 16;
    const uint4 x = *(const uint4*)(base[kv] + from[r0 + row] * p.row_bytes + off);
    *(uint4*)(base[kv] + holes[r0 + row] * p.row_bytes + off) = x;
  }
}

namespace {

int evict_check(const InfernoEvict* e) {
  if (!e) return set_error(INFERNO_EINVAL, "cache_evict: null parameters");
  if (e->struct_size != (int)sizeof(InfernoEvict))
    return set_error(INFERNO_EINVAL, "cache_evict: struct_size %d, expected %d", e->struct_size,
                     (int)sizeof(InfernoEvict));
  const int es = longctx_type_size(e->type);
  if (!es) return set_error(INFERNO_EINVAL, "cache_evict: type %d is not F32, F16 or BF16", e->type);
  if (e->batch < 0 || e->n_kv_heads < 1 || e->head_dim < 1 || e->max_len < 0 || e->n_kv_heads > 65535 ||
      (long long)e->batch * e->n_kv_heads > 65535)
    return set_error(INFERNO_EINVAL, "cache_evict: bad sizes (batch %d, %d KV heads of %d, max_len %d)", e->batch,
                     e->n_kv_heads, e->head_dim, e->max_len);
  if ((long long)e->head_dim * es % 16 || e->head_dim > 8192)
    return set_error(INFERNO_EINVAL, "cache_evict: head_dim %d is not a multiple of 16 bytes or above 8192",
                     e->head_dim);
  if (e->budget < 1) return set_error(INFERNO_EINVAL, "cache_evict: budget %d", e->budget);
  if (e->n_sink < 0 || e->n_recent < 0 || (long long)e->n_sink + e->n_recent > e->budget)
    return set_error(INFERNO_EINVAL, "cache_evict: n_sink %d + n_recent %d exceed the budget %d", e->n_sink,
                     e->n_recent, e->budget);
  if (e->reserved) return set_error(INFERNO_EINVAL, "cache_evict: reserved must be 0");
  return 0;
}

int evict_max_moves(const InfernoEvict* e) { return std::max(0, std::min(e->budget, e->max_len - e->budget)); }

int64_t evict_workspace(const InfernoEvict* e) {
  const int64_t n = (int64_t)e->batch * e->n_kv_heads;
  return ((n * 4 + 255) / 256 + 1) * 256 + n * 2 * evict_max_moves(e) * 4;
}

}  // namespace
}  // namespace inf

using namespace inf;

extern "C" int64_t inferno_cache_evict_workspace(const InfernoEvict* e) {
  const int rc = evict_check(e);
  return rc ? rc : evict_workspace(e);
}

extern "C" int inferno_cache_evict(const InfernoEvict* e, void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = evict_check(e);
  if (rc) return rc;
  if (e->batch == 0) return 0;
  if (!e->k_cache || !e->v_cache || !e->scores || !e->slot_pos || !e->lens || !e->next_pos || !e->scores_out ||
      !e->slot_pos_out || !e->lens_out)
    return set_error(INFERNO_EINVAL, "cache_evict: null pointer");
  const int es = longctx_type_size(e->type);
  const long long row = (long long)e->n_kv_heads * e->head_dim;
  if (e->batch > 1 && e->seq_stride < row * e->max_len)
    return set_error(INFERNO_EINVAL, "cache_evict: seq_stride %lld is less than a slice of %d rows",
                     (long long)e->seq_stride, e->max_len);
  if (e->score_stride < e->max_len && (long long)e->batch * e->n_kv_heads > 1)
    return set_error(INFERNO_EINVAL, "cache_evict: score_stride %lld is less than max_len %d",
                     (long long)e->score_stride, e->max_len);
  if (e->seq_stride * es % 16 || (uintptr_t)e->k_cache % 16 || (uintptr_t)e->v_cache % 16)
    return set_error(INFERNO_EINVAL, "cache_evict: caches and seq_stride must be multiples of 16 bytes");
  if (((uintptr_t)e->scores | (uintptr_t)e->slot_pos | (uintptr_t)e->lens | (uintptr_t)e->next_pos |
       (uintptr_t)e->scores_out | (uintptr_t)e->slot_pos_out | (uintptr_t)e->lens_out) % 4)
    return set_error(INFERNO_EINVAL, "cache_evict: a pointer is not a multiple of 4 bytes");
  if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < evict_workspace(e))
    return set_error(INFERNO_EINVAL, "cache_evict: workspace of %lld bytes, %lld needed (256-byte aligned)",
                     (long long)workspace_bytes, (long long)evict_workspace(e));
  if ((rc = longctx_check_device(e->k_cache, "cache_evict"))) return rc;
  EvictParams p{};
  p.kc = (uint8_t*)e->k_cache;
  p.vc = (uint8_t*)e->v_cache;
  p.seq_bytes = e->batch > 1 ? e->seq_stride * es : 0;
  p.row_bytes = row * es;
  p.head_bytes = e->head_dim * es;
  p.scores = e->scores;
  p.pos = e->slot_pos;
  p.lens = e->lens;
  p.next_pos = e->next_pos;
  p.scores_out = e->scores_out;
  p.pos_out = e->slot_pos_out;
  p.lens_out = e->lens_out;
  p.stride = e->score_stride;
  p.batch = e->batch;
  p.nkv = e->n_kv_heads;
  p.max_len = e->max_len;
  p.budget = e->budget;
  p.n_sink = e->n_sink;
  p.n_recent = e->n_recent;
  p.max_moves = evict_max_moves(e);
  const int n = e->batch * e->n_kv_heads;
  p.counts = (int*)workspace;
  p.lists = (int*)((char*)workspace + ((size_t)n * 4 + 255) / 256 * 256);
  cudaStream_t st = (cudaStream_t)stream;
  evict_select_kernel<<<n, EV_THREADS, 0, st>>>(p);
  cudaError_t err = cudaGetLastError();
  if (err == cudaSuccess) {
    const int rows = std::max(1, EV_MOVE_THREADS * 4 / (2 * p.head_bytes / 16));
    const int bx = std::max(1, (p.max_moves + rows - 1) / rows);
    evict_move_kernel<<<dim3(bx, n), EV_MOVE_THREADS, 0, st>>>(p, rows);
    err = cudaGetLastError();
  }
  return err == cudaSuccess ? 0 : set_error(INFERNO_ECUDA, "cache_evict launch: %s", cudaGetErrorString(err));
}
