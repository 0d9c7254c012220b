// Eviction of cache rows by gathered attention weight (inferno_cache_evict).
//
// One thread-block cluster per (sequence, KV head); each CTA owns a consecutive
// part of the rows.  The rank key is the score as an order-preserving 32-bit
// integer, in two classes (rows kept always come first); it is read once into
// shared memory.  The budget-th largest key is found by a radix select of four
// 8-bit digits: every CTA counts its own rows, reads the others' counts through
// distributed shared memory and finds the digit for itself; it ends early where all
// rows of the border's bin stay.  (Digits of 11 bits
// save a barrier and cost eight times the remote reads, which are what a pass
// waits for: 10 us a pass measured with 8 CTAs, 1 us with 8 bits.)
// Ties at that key (or in that bin) go to the lowest rows.  Which rows stay is then a bitmap, so
// ranks are bit counts: the i-th kept row behind the budget goes into the i-th
// hole before it.  The two lists have equal lengths and no row is both read and
// written, so the CTAs of the cluster move K and V in any order.
//
// Bound: the bytes of the rows that move (read and written), after a chain of
// up to seven cluster barriers (four digits, the first once more where the rows kept
// always exceed the budget, the ties, the lists) that few rows cannot hide.
#include <algorithm>
#include <cooperative_groups.h>
#include "internal.h"
#include "common.cuh"
#include "longctx.h"
#include "../../include/inferno_b200.h"

namespace inf {

namespace cg = cooperative_groups;

constexpr int EV_THREADS = 1024;
constexpr int EV_WARPS = EV_THREADS / 32;
constexpr int EV_MOVE_THREADS = 256;
constexpr int EV_BINS = 256;
constexpr int EV_MAX_CLUSTER = 16;         // B200's largest, above the portable 8
constexpr int EV_MAX_LEN = 1000000;         // a sixteenth has fewer than 2^16 rows (counts), and its bitmaps fit shared memory
constexpr int EV_SMEM = 200 * 1024;

struct EvictParams {
  uint8_t *kc, *vc;
  long long seq_bytes, row_bytes;     // bytes between slices; between rows of one KV head
  int head_bytes;
  const float* scores;
  const int* pos;
  const int *lens, *next_pos;
  float* scores_out;
  int *pos_out, *lens_out;            // lens_out null: written by evict_move_kernel
  long long stride;                   // entries between (sequence, KV head) rows of scores / pos
  int nkv, max_len, budget, n_sink, n_recent, max_moves;
  int words;                          // 32-row words a CTA's part may have
  int cached;                         // keys held in shared memory
  int* lists;                         // [batch * nkv][2][max_moves]: holes, sources
  int* counts;                        // [batch * nkv] rows to move; null: the clusters move K and V themselves
};

// larger is kept first; NaN below everything; -0 equal to 0
__device__ __forceinline__ uint32_t ev_key(float s) { return s != s ? 0u : float_ordered(s + 0.0f); }

// what a CTA's peers read
struct EvShared {
  uint32_t hist[2][EV_BINS / 2];      // counts of a digit, two 16-bit ones per word: half the bytes to read
  int4 border;                        // ties before / behind the budget, other rows to leave before it / to keep behind it
  int always;                         // rows kept always
  // the CTA's own
  int2 warp_sums[EV_WARPS], sum;
  int bin_sums[EV_BINS / 64];
  int digit, need, in_bin;             // in_bin: rows in the digit's bin
};

// exclusive sums of x and y over the CTA in thread order; the CTA's in sum_x, sum_y
__device__ __forceinline__ void ev_scan(EvShared& s, int& x, int& y, int& sum_x, int& sum_y) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int a = x, b = y;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, a, o), v = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) a += u, b += v;
  }
  __syncthreads();                     // the last call's sums are read
  if (lane == 31) s.warp_sums[warp] = make_int2(a, b);
  __syncthreads();
  if (warp == 0) {                     // EV_WARPS = 32
    const int2 w = s.warp_sums[lane];
    int c = w.x, d = w.y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, c, o), v = __shfl_up_sync(0xffffffffu, d, o);
      if (lane >= o) c += u, d += v;
    }
    s.warp_sums[lane] = make_int2(c - w.x, d - w.y);
    if (lane == 31) s.sum = make_int2(c, d);
  }
  __syncthreads();
  const int2 base = s.warp_sums[warp], all = s.sum;
  x = base.x + a - x;
  y = base.y + b - y;
  sum_x = all.x, sum_y = all.y;
}

__global__ void __launch_bounds__(EV_THREADS, 1) evict_kernel(const __grid_constant__ EvictParams p) {
  pdl_trigger();                              // evict_move_kernel may take its places on the idle SMs
  cg::cluster_group cluster = cg::this_cluster();
  const int nc = cluster.num_blocks(), c = cluster.block_rank();
  const int bh = blockIdx.x / nc, b = bh / p.nkv, h = bh - b * p.nkv;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  __shared__ EvShared sh;
  extern __shared__ uint32_t ev_dyn[];
  uint32_t* always = ev_dyn;                  // bit per row of the part: kept always
  uint32_t* tie = always + p.words;           // key equal to the border in its leading digits
  uint32_t* keep = tie + p.words;
  int* base_h = (int*)(keep + p.words);       // holes / sources before a word
  int* base_s = base_h + p.words;
  uint32_t* skey = (uint32_t*)(base_s + p.words);

  const int next = p.next_pos[b], len = max(0, min(p.lens[b], p.max_len));
  if (p.lens_out && h == 0 && c == 0 && t == 0) p.lens_out[b] = min(len, p.budget);
  const float* sc = p.scores + bh * p.stride;
  const int* ps = p.pos + bh * p.stride;
  float* so = p.scores_out + bh * p.stride;
  int* po = p.pos_out + bh * p.stride;
  if (len <= p.budget) {                      // the whole cluster leaves
    if (p.counts && c == 0 && t == 0) p.counts[bh] = 0;
    for (int j = c * EV_THREADS + t; j < len; j += nc * EV_THREADS) {
      if (so != sc) so[j] = sc[j];
      if (po != ps) po[j] = ps[j];
    }
    return;
  }
  auto sync_all = [&] {
    if (nc == 1) __syncthreads();
    else cluster.sync();
  };
  // this CTA's rows [j0, j0 + n), in words of 32
  const int words_all = (len + 31) >> 5, wpc = (words_all + nc - 1) / nc;
  const int j0 = min(c * wpc, words_all) * 32, n = min(len - j0, wpc * 32), nw = (n + 31) >> 5;
  const int recent_from = (int)max(-2147483648ll, (long long)next - p.n_recent);
  if (t < EV_BINS) (&sh.hist[0][0])[t] = 0;
  if (t == 0) sh.always = 0;
  __syncthreads();
  auto key_of = [&](int i) { return p.cached ? skey[i] : ev_key(sc[j0 + i]); };

  // ---- read, and the first digit of the rows not kept always -------------------
  int n_always = 0;
  for (int w0 = warp; w0 < nw; w0 += 4 * EV_WARPS) {
    float s[4];
    int at[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = (w0 + u * EV_WARPS) * 32 + lane;
      s[u] = i < n ? sc[j0 + i] : 0.f;
      at[u] = i < n ? ps[j0 + i] : 0;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int w = w0 + u * EV_WARPS, i = w * 32 + lane;
      if (w >= nw) break;
      const uint32_t k = ev_key(s[u]);
      const bool in = i < n, al = in && (at[u] < p.n_sink || at[u] >= recent_from);
      const uint32_t m = __ballot_sync(0xffffffffu, al);
      if (lane == 0) always[w] = m;
      n_always += __popc(m);
      if (p.cached) skey[i] = k;
      if (in && !al) atomicAdd(&sh.hist[0][k >> 25], 1u << (k >> 24 & 1) * 16);
    }
  }
  if (lane == 0 && n_always) atomicAdd(&sh.always, n_always);

  // ---- radix select ---------------------------------------------------------------
  // the class the border lies in: the others, or the rows kept always should they
  // exceed the budget (the first digit is then counted again)
  bool among_always = false, recount = false;
  int need = 0, buf = 0, shift = 24;
  uint32_t prefix = 0;
  while (shift >= 0) {
    if (shift < 24 || recount) {
      for (int i = t; i < n; i += EV_THREADS) {
        const uint32_t k = key_of(i);
        if ((((always[i >> 5] >> (i & 31)) & 1) != 0) == among_always && (shift == 24 || (k >> (shift + 8)) == prefix))
          atomicAdd(&sh.hist[buf][(k >> (shift + 1)) & 127], 1u << (k >> shift & 1) * 16);
      }
    }
    sync_all();
    if (shift == 24 && !recount) {
      int al = lane < nc ? *cluster.map_shared_rank(&sh.always, lane) : 0;
      al = __reduce_add_sync(0xffffffffu, al);
      need = p.budget - al;
      if (need < 0) {
        need = p.budget;
        among_always = recount = true;
        buf = 1;
        continue;
      }
    }
    // thread t: bins 2 t and 2 t + 1 of the whole cluster, and what lies in the bins
    // above; the digit's bin holds the need-th largest key (need 0: no row of this
    // class)
    int lo = 0, hi = 0, above = 0;
    if (t < EV_BINS / 2) {
      if (nc == 1) {
        lo = sh.hist[buf][t] & 0xffff;
        hi = sh.hist[buf][t] >> 16;
      } else {
        uint32_t x[EV_MAX_CLUSTER];           // all loads in flight
#pragma unroll
        for (int r = 0; r < EV_MAX_CLUSTER; ++r) x[r] = r < nc ? cluster.map_shared_rank(&sh.hist[buf][0], r)[t] : 0u;
#pragma unroll
        for (int r = 0; r < EV_MAX_CLUSTER; ++r) lo += x[r] & 0xffff, hi += x[r] >> 16;
      }
      sh.hist[buf ^ 1][t] = 0;                // free: its readers passed the barrier above
      above = lo + hi;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_down_sync(0xffffffffu, above, o);
        if (lane + o < 32) above += u;
      }
      if (lane == 0) sh.bin_sums[warp] = above;
    }
    if (t == EV_BINS) sh.digit = 255, sh.need = sh.in_bin = 0;
    __syncthreads();
    if (t < EV_BINS / 2) {
      above -= lo + hi;
#pragma unroll
      for (int w = 1; w < EV_BINS / 64; ++w)
        if (w > warp) above += sh.bin_sums[w];
      if (above < need && above + hi >= need) sh.digit = 2 * t + 1, sh.need = need - above, sh.in_bin = hi;
      above += hi;
      if (above < need && above + lo >= need) sh.digit = 2 * t, sh.need = need - above, sh.in_bin = lo;
    }
    __syncthreads();
    const int digit = sh.digit;
    need = sh.need;
    prefix = (prefix << 8) | (uint32_t)digit;
    buf ^= 1;
    shift -= 8;
    if (sh.in_bin == need) break;             // all of the bin: the digits below do not matter (mostly the last one)
  }
  const int low = shift + 8;                  // bits of the digits left out

  // ---- bitmaps: kept for certain, and ties at the border ------------------------------
  for (int w = warp; w < nw; w += EV_WARPS) {
    const int i = w * 32 + lane;
    const uint32_t k = i < n ? key_of(i) : 0u;
    const bool al = (always[w] >> lane) & 1, in_class = i < n && al == among_always;
    const uint32_t m_tie = __ballot_sync(0xffffffffu, in_class && k >> low == prefix);
    const uint32_t m_keep = __ballot_sync(0xffffffffu, i < n && (in_class ? k >> low > prefix : al));
    if (lane == 0) tie[w] = m_tie, keep[w] = m_keep;
  }
  __syncthreads();
  // thread t owns words [w_lo, w_hi); front(w): rows of word w before the budget
  const int wpt = (nw + EV_THREADS - 1) / EV_THREADS, w_lo = min(nw, t * wpt), w_hi = min(nw, w_lo + wpt);
  auto valid = [&](int w) { return n - w * 32 >= 32 ? 0xffffffffu : (1u << (n - w * 32)) - 1; };
  auto front = [&](int w) {
    const int m = p.budget - (j0 + w * 32);
    return m >= 32 ? 0xffffffffu : m <= 0 ? 0u : (1u << m) - 1;
  };
  // counts of a part fit 16 bits: two per scanned word
  int tf = 0, ls = 0, sum_tf, sum_ls;        // ties, and those in front; leave in front, stay behind
  for (int w = w_lo; w < w_hi; ++w) {
    const uint32_t f = front(w);
    tf += __popc(tie[w]) | __popc(tie[w] & f) << 16;
    ls += __popc(~(keep[w] | tie[w]) & valid(w) & f) | __popc(keep[w] & ~f) << 16;
  }
  ev_scan(sh, tf, ls, sum_tf, sum_ls);
  int ties = tf & 0xffff;
  const int sum = sum_tf & 0xffff, sum_front = (uint32_t)sum_tf >> 16;
  const int sum_leave = sum_ls & 0xffff, sum_stay = (uint32_t)sum_ls >> 16;
  if (t == 0) sh.border = make_int4(sum_front, sum - sum_front, sum_leave, sum_stay);
  sync_all();
  // lane r: CTA r's part.  Its ties are kept as far as `need` reaches after those
  // of the CTAs before it, the ones before the budget first
  int holes, srcs, moves;
  {
    const int4 x = lane < nc ? *cluster.map_shared_rank(&sh.border, lane) : make_int4(0, 0, 0, 0);
    int before = x.x + x.y;
#pragma unroll
    for (int o = 1; o < EV_MAX_CLUSTER; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += u;
    }
    before -= x.x + x.y;
    const int kept = max(0, min(need - before, x.x + x.y)), kept_front = min(kept, x.x);
    int hr = x.z + x.x - kept_front, sr = x.w + kept - kept_front;      // holes and sources of CTA r
    moves = __reduce_add_sync(0xffffffffu, sr);
    holes = __reduce_add_sync(0xffffffffu, lane < c ? hr : 0);
    srcs = __reduce_add_sync(0xffffffffu, lane < c ? sr : 0);
    ties += __shfl_sync(0xffffffffu, before, c);                       // ties before this thread's words
  }
  int nh = 0, ns = 0;
  for (int w = w_lo; w < w_hi; ++w) {
    uint32_t m = tie[w], k = keep[w];
    for (; m && ties < need; m &= m - 1, ++ties) k |= m & (0u - m);
    ties += __popc(m);
    keep[w] = k;
    nh += base_h[w] = __popc(~k & valid(w) & front(w));
    ns += base_s[w] = __popc(k & ~front(w));
  }
  int sum_h, sum_s;
  ev_scan(sh, nh, ns, sum_h, sum_s);
  holes += nh, srcs += ns;
  for (int w = w_lo; w < w_hi; ++w) {
    const int x = base_h[w], y = base_s[w];
    base_h[w] = holes, base_s[w] = srcs;
    holes += x, srcs += y;
  }
  __syncthreads();

  // ---- the lists, and the rows that stay in place -----------------------------------
  int* hole_list = p.lists + (long long)bh * 2 * p.max_moves;
  int* src_list = hole_list + p.max_moves;
  const uint32_t lt = (1u << lane) - 1;
  const bool copy = so != sc || po != ps;
  for (int w0 = warp; w0 < nw; w0 += 4 * EV_WARPS) {
    float x[4];
    int at[4];
    if (copy) {                               // four words' loads in flight
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int w = w0 + u * EV_WARPS, i = w * 32 + lane;
        const bool stays = w < nw && j0 + i < p.budget && ((keep[min(w, nw - 1)] >> lane) & 1);
        x[u] = stays ? sc[j0 + i] : 0.f;
        at[u] = stays ? ps[j0 + i] : 0;
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int w = w0 + u * EV_WARPS, i = w * 32 + lane, j = j0 + i;
      if (w >= nw) break;
      const bool kept = (keep[w] >> lane) & 1, front = j < p.budget;
      const uint32_t m_h = __ballot_sync(0xffffffffu, i < n && front && !kept);
      const uint32_t m_s = __ballot_sync(0xffffffffu, !front && kept);
      if ((m_h >> lane) & 1) hole_list[base_h[w] + __popc(m_h & lt)] = j;
      if ((m_s >> lane) & 1) src_list[base_s[w] + __popc(m_s & lt)] = j;
      if (copy && front && kept) so[j] = x[u], po[j] = at[u];
    }
  }
  sync_all();                             // lists complete; also the last read of a peer's shared memory

  // ---- move ---------------------------------------------------------------------------
  for (int i = c * EV_THREADS + t; i < moves; i += nc * EV_THREADS) {
    const int from = src_list[i], to = hole_list[i];
    so[to] = sc[from];
    po[to] = ps[from];
  }
  if (p.counts) {
    if (c == 0 && t == 0) p.counts[bh] = moves;
    return;
  }
  const int vecs = p.head_bytes / 16;         // 16-byte pieces of a K row; as many of the V row
  uint8_t* kb = p.kc + b * p.seq_bytes + (long long)h * p.head_bytes;
  uint8_t* vb = p.vc + b * p.seq_bytes + (long long)h * p.head_bytes;
  const int iters = (2 * vecs + 31) / 32, stride = nc * EV_WARPS, first = c * EV_WARPS + warp;
  const int mine = moves > first ? (moves - first + stride - 1) / stride : 0;
  constexpr int U = 6;                        // pieces in flight per lane
  int m = 0, it = 0;                          // move and piece of the next unit
  for (int u0 = 0; u0 < mine * iters; u0 += U) {
    uint4 x[U];
    int to[U], piece[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      piece[u] = it * 32 + lane;
      to[u] = -1;
      if (m < mine && piece[u] < 2 * vecs) {
        const int at = first + m * stride;
        const uint8_t* base = piece[u] < vecs ? kb + piece[u] * 16 : vb + (piece[u] - vecs) * 16;
        to[u] = hole_list[at];
        x[u] = *(const uint4*)(base + src_list[at] * p.row_bytes);
      }
      if (++it == iters) it = 0, ++m;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (to[u] >= 0) *(uint4*)((piece[u] < vecs ? kb + piece[u] * 16 : vb + (piece[u] - vecs) * 16) + to[u] * p.row_bytes) = x[u];
  }
}

// After evict_kernel: lens_out in place, once every cluster has read lens, and K and
// V where there are too few (sequence, KV head) clusters to fill the GPU.
__global__ void __launch_bounds__(EV_MOVE_THREADS) evict_move_kernel(const __grid_constant__ EvictParams p, int* lens, int rows_per_block) {
  const int bh = blockIdx.y, b = bh / p.nkv, h = bh - b * p.nkv;
  pdl_wait();
  if (lens && blockIdx.x == 0 && h == 0 && threadIdx.x == 0) lens[b] = min(max(0, min(lens[b], p.max_len)), p.budget);
  if (!p.counts) return;
  const int r0 = blockIdx.x * rows_per_block, n = min(p.counts[bh] - r0, rows_per_block);
  const int* holes = p.lists + (long long)bh * 2 * p.max_moves + r0;
  const int* from = holes + p.max_moves;
  const int vecs = p.head_bytes / 16;
  uint8_t* kb = p.kc + b * p.seq_bytes + (long long)h * p.head_bytes;
  uint8_t* vb = p.vc + b * p.seq_bytes + (long long)h * p.head_bytes;
  constexpr int U = 8;
  for (int i0 = threadIdx.x; i0 < n * 2 * vecs; i0 += U * EV_MOVE_THREADS) {
    uint4 x[U];
    uint8_t* dst[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * EV_MOVE_THREADS, row = i / (2 * vecs), piece = i - row * 2 * vecs;
      dst[u] = nullptr;
      if (row >= n) continue;
      uint8_t* base = piece < vecs ? kb + piece * 16 : vb + (piece - vecs) * 16;
      dst[u] = base + holes[row] * p.row_bytes;
      x[u] = *(const uint4*)(base + from[row] * p.row_bytes);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (dst[u]) *(uint4*)dst[u] = x[u];
  }
}

namespace {

int evict_check(const InfernoEvict* e) {
  if (!e) return set_error(INFERNO_EINVAL, "cache_evict: null parameters");
  if (e->struct_size && e->struct_size != (int)sizeof(InfernoEvict))
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
  if (e->max_len > EV_MAX_LEN)
    return set_error(INFERNO_EINVAL, "cache_evict: max_len %d is above %d", e->max_len, EV_MAX_LEN);
  if (e->budget < 1) return set_error(INFERNO_EINVAL, "cache_evict: budget %d", e->budget);
  if (e->n_sink < 0 || e->n_recent < 0 || (long long)e->n_sink + e->n_recent > e->budget)
    return set_error(INFERNO_EINVAL, "cache_evict: n_sink %d + n_recent %d exceed the budget %d", e->n_sink,
                     e->n_recent, e->budget);
  if (e->reserved) return set_error(INFERNO_EINVAL, "cache_evict: reserved must be 0");
  return 0;
}

int evict_max_moves(const InfernoEvict* e) { return std::max(0, std::min(e->budget, e->max_len - e->budget)); }

int64_t evict_workspace(const InfernoEvict* e) {
  return (int64_t)e->batch * e->n_kv_heads * (2 * (int64_t)evict_max_moves(e) + 1) * 4 + 256;
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
  if ((rc = longctx_check_device({e->k_cache, e->v_cache, e->scores, e->slot_pos, e->lens, e->next_pos, e->scores_out,
                                  e->slot_pos_out, e->lens_out, workspace}, "cache_evict")))
    return rc;
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
  p.nkv = e->n_kv_heads;
  p.max_len = e->max_len;
  p.budget = e->budget;
  p.n_sink = e->n_sink;
  p.n_recent = e->n_recent;
  p.max_moves = evict_max_moves(e);
  p.lists = (int*)workspace;
  if (e->lens_out == e->lens) p.lens_out = nullptr;
  // CTAs per (sequence, KV head), up to 16: one per 4096 rows to rank (fewer do not
  // pay for the cluster's barriers, of which one CTA has none) or per 512 KB to move.
  // All clusters have to run at once, an SM per CTA (a second round of them costs a
  // whole ranking): 35 clusters of 4 fit, 16 of 8 and 7 of 16 at best, so clusters of
  // 8 and 16 are kept to 64 CTAs (8 heads of 54775 fp32 rows: 39 us with 8 CTAs each,
  // 65 with 16)
  const int n = e->batch * e->n_kv_heads;
  int dev = 0;
  INF_CUDA_TRY(cudaGetDevice(&dev));
  int nc = 1;
  while (nc < EV_MAX_CLUSTER && n * nc * 2 <= (nc >= 4 ? 64 : 128) &&
         (e->max_len >= nc * 2 * 4096 || 4ll * p.max_moves * p.head_bytes >= nc * 2 * (512ll << 10)))
    nc *= 2;
  auto smem_of = [&](int ctas, bool cached) {
    const long long words = ((e->max_len + 31) / 32 + ctas - 1) / ctas;
    return words * 4 * (5 + (cached ? 32 : 0));
  };
  while (nc < EV_MAX_CLUSTER && smem_of(nc, true) > EV_SMEM) nc *= 2;
  p.cached = smem_of(nc, true) <= EV_SMEM;
  p.words = ((e->max_len + 31) / 32 + nc - 1) / nc;
  const size_t smem = smem_of(nc, p.cached);
  // much to move by less than half of the SMs: a second kernel over the whole GPU
  // moves K and V (4 heads of 62898 fp32 rows of 128 to 14946: 105 us with 32 CTAs
  // alone, 45 with it)
  const bool spread = n * nc * 2 < num_sms(dev) && 4ll * p.max_moves * p.head_bytes > nc * (512ll << 10);
  if (spread) p.counts = (int*)workspace + (long long)n * 2 * p.max_moves;
  cudaStream_t st = (cudaStream_t)stream;
  static DeviceOnce once;
  cudaError_t err = once.run([] {
    const cudaError_t a = cudaFuncSetAttribute(evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_SMEM);
    return a == cudaSuccess ? cudaFuncSetAttribute(evict_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) : a;
  });
  if (err == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n * nc));
    cfg.blockDim = dim3(EV_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = nc;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    err = cudaLaunchKernelEx(&cfg, evict_kernel, p);
  }
  if (err == cudaSuccess && (spread || !p.lens_out)) {
    const int rows = std::max(1, (16 << 10) / p.head_bytes);         // 32 KB of K and V: one piece in flight each
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(spread ? (p.max_moves + rows - 1) / rows : 1), (unsigned)n);
    cfg.blockDim = dim3(EV_MOVE_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    err = cudaLaunchKernelEx(&cfg, evict_move_kernel, p, p.lens_out ? nullptr : e->lens_out, rows);
  }
  return err == cudaSuccess ? 0 : set_error(INFERNO_ECUDA, "cache_evict launch: %s", cudaGetErrorString(err));
}
