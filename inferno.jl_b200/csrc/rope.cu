// Rotary positions of q and k with the append of k and v to cache rows
// (inferno_rope).
//
// A pair (a, b) of a head becomes (a cos - b sin, a sin + b cos) with the angle
// positions[t] * f_i.  A block takes TB tokens (and a slice of their heads): its
// threads first put cos and sin of the tokens' angles into shared memory, once
// for all heads, then stream the heads through registers, one 16-byte vector
// (two for the half layout, whose pairs lie rope_dim / 2 apart) per item.
//
// Angles: f_i / (2 pi) is a double, so positions[t] * f_i / (2 pi) has the turn
// exact to 2^-52 of itself; the whole turns are dropped in double and the rest,
// at most half a turn, goes to sincospi in fp32.  The error is that of an fp32
// angle below pi (about 1e-7) at any position.
//
// Bound: bytes, each value read and written once.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <cuda_bf16.h>
#include "internal.h"
#include "common.cuh"
#include "longctx.h"
#include "../../include/inferno_b200.h"

namespace inf {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_MAX_PAIRS = 256;

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery, "Division by
// invariant integers using multiplication", 1994)
struct FastDiv {
  uint32_t d, mul, shift;
  __host__ FastDiv(uint32_t div = 1) : d(div) {
    shift = 0;
    while ((1ull << shift) < d) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

struct RopeParams {
  const void *q, *k, *v;
  void *qo, *ko, *vo;
  long long qs, ks, vs, qos, kos, vos;   // elements between token rows
  const int *positions, *slots;
  const float* freq_factors;
  int n_tokens, n_rows, head_dim, rope_dim;
  int tb;                                // tokens per block
  uint32_t items;                        // items of one token (q, then k, then v)
  uint32_t q_items, k_items;             // items of q alone, of q and k
  uint32_t slice;                        // items of one block (over its tb tokens)
  FastDiv by_items, by_head;             // items per token; items per head of q and k
  uint32_t rot_items;                    // items of a head that are rotated
  float gain, sign;                      // factor of cos and sin; -1: rotate back
  double turns[ROPE_MAX_PAIRS];          // f_i / (2 pi), without freq_factors
};

template <typename T>
__device__ __forceinline__ float to_f(T x) {
  if constexpr (std::is_same_v<T, float>) return x;
  else if constexpr (std::is_same_v<T, __half>) return __half2float(x);
  else return __bfloat162float(x);
}
template <typename T>
__device__ __forceinline__ T from_f(float x) {
  if constexpr (std::is_same_v<T, float>) return x;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T x[V];
};

// V: elements of one access (the widest that sizes, strides and pointers
// allow).  ILV: interleaved pairs; one item then holds whole pairs.
template <typename T, int V, bool ILV>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(const __grid_constant__ RopeParams p) {
  extern __shared__ float2 cs[];                     // [tb][rope_dim / 2] (cos, sin)
  constexpr int RV = ILV && V < 2 ? 2 : V;           // values of one rotated vector
  constexpr int NP = ILV ? RV / 2 : RV;              // pairs of one rotated item
  using Vt = Vec<T, V>;
  const int half = p.rope_dim >> 1;
  const int t0 = blockIdx.x * p.tb, nt = min(p.tb, p.n_tokens - t0);
  for (int i = threadIdx.x; i < nt * half; i += ROPE_THREADS) {
    const int t = i / half, c = i - t * half;
    double turn = p.turns[c];
    if (p.freq_factors) turn /= (double)__ldg(p.freq_factors + c);
    turn *= (double)__ldg(p.positions + t0 + t);
    turn -= rint(turn);
    float sn, cn;
    sincospif(2.0f * (float)turn, &sn, &cn);
    cs[i] = make_float2(cn * p.gain, sn * p.gain * p.sign);
  }
  __syncthreads();
  const uint32_t end = min((blockIdx.y + 1) * p.slice, (uint32_t)nt * p.items);
  constexpr int U = 2;                               // items in flight per thread
  for (uint32_t e0 = blockIdx.y * p.slice + threadIdx.x; e0 < end; e0 += U * ROPE_THREADS) {
    alignas(16) T a[U][RV];
    alignas(16) T b[U][RV];
    T* dst[U];
    int pair[U];                                     // first pair, or -1: copied
#pragma unroll
    for (int u = 0; u < U; ++u) {
      dst[u] = nullptr;
      const uint32_t e = e0 + u * ROPE_THREADS;
      if (e >= end) continue;
      const uint32_t tl = p.by_items.div(e);
      uint32_t it = e - tl * p.items;
      const int t = t0 + (int)tl;
      const T* src;
      long long row = t;
      if (it >= p.q_items && p.slots) {
        row = __ldg(p.slots + t);
        if (row < 0 || row >= p.n_rows) continue;
      }
      if (it >= p.k_items) {                         // v: copied whole
        it -= p.k_items;
        src = (const T*)p.v + (long long)t * p.vs + (long long)it * V;
        dst[u] = (T*)p.vo + row * p.vos + (long long)it * V;
        pair[u] = -1;
      } else {
        const bool isq = it < p.q_items;
        if (!isq) it -= p.q_items;
        const uint32_t h = p.by_head.div(it), j = it - h * p.by_head.d;
        const bool rot = j < p.rot_items;
        const long long off = (long long)h * p.head_dim +
                              (rot ? (long long)j * RV : (long long)p.rope_dim + (long long)(j - p.rot_items) * V);
        src = isq ? (const T*)p.q + (long long)t * p.qs + off : (const T*)p.k + (long long)t * p.ks + off;
        dst[u] = isq ? (T*)p.qo + row * p.qos + off : (T*)p.ko + row * p.kos + off;
        pair[u] = rot ? (int)(tl * half + j * NP) : -1;
      }
      if (pair[u] < 0) {
        *(Vt*)a[u] = *(const Vt*)src;
      } else {
#pragma unroll
        for (int i = 0; i < RV; i += V) *(Vt*)(a[u] + i) = *(const Vt*)(src + i);
        if constexpr (!ILV) *(Vt*)b[u] = *(const Vt*)(src + half);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!dst[u]) continue;
      if (pair[u] < 0) {
        *(Vt*)dst[u] = *(const Vt*)a[u];
        continue;
      }
      const float2* w = cs + pair[u];
      if constexpr (ILV) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const float2 c = w[i];
          const float x = to_f(a[u][2 * i]), y = to_f(a[u][2 * i + 1]);
          a[u][2 * i] = from_f<T>(x * c.x - y * c.y);
          a[u][2 * i + 1] = from_f<T>(x * c.y + y * c.x);
        }
#pragma unroll
        for (int i = 0; i < RV; i += V) *(Vt*)(dst[u] + i) = *(const Vt*)(a[u] + i);
      } else {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const float2 c = w[i];
          const float x = to_f(a[u][i]), y = to_f(b[u][i]);
          a[u][i] = from_f<T>(x * c.x - y * c.y);
          b[u][i] = from_f<T>(x * c.y + y * c.x);
        }
        *(Vt*)dst[u] = *(const Vt*)a[u];
        *(Vt*)(dst[u] + half) = *(const Vt*)b[u];
      }
    }
  }
}

namespace {

// `count` rows of `width` bytes, `stride` bytes apart
struct Rows {
  const char* p;
  long long stride, width, count;
  __int128 begin() const { return (__int128)(uintptr_t)p; }
  __int128 end() const { return begin() + (__int128)(count - 1) * stride + width; }
};
// whether a row of a may share a byte with a row of b: no when the ranges are
// apart, or when equal strides leave every row of the one between rows of the
// other (q, k and v of one fused row); yes wherever that is not certain
bool rows_overlap(const Rows& a, const Rows& b) {
  if (!a.p || !b.p || a.count <= 0 || b.count <= 0) return false;
  if (a.end() <= b.begin() || b.end() <= a.begin()) return false;
  if (a.stride != b.stride || a.stride <= 0) return true;
  long long d = (long long)((b.begin() - a.begin()) % a.stride);
  if (d < 0) d += a.stride;
  return !(d >= a.width && a.stride - d >= b.width);
}

template <typename T, int V>
cudaError_t rope_launch_v(const RopeParams& p, bool ilv, dim3 grid, size_t smem, cudaStream_t st) {
  if (ilv)
    rope_kernel<T, V, true><<<grid, ROPE_THREADS, smem, st>>>(p);
  else
    rope_kernel<T, V, false><<<grid, ROPE_THREADS, smem, st>>>(p);
  return cudaGetLastError();
}
template <typename T>
cudaError_t rope_launch(const RopeParams& p, int vec, bool ilv, dim3 grid, size_t smem, cudaStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return rope_launch_v<T, 8>(p, ilv, grid, smem, st);
  if (vec >= 4) return rope_launch_v<T, 4>(p, ilv, grid, smem, st);
  if (vec == 2) return rope_launch_v<T, 2>(p, ilv, grid, smem, st);
  return rope_launch_v<T, 1>(p, ilv, grid, smem, st);
}

}  // namespace
}  // namespace inf

using namespace inf;

extern "C" int inferno_rope(const InfernoRope* r, void* stream) {
  if (!r) return set_error(INFERNO_EINVAL, "rope: null parameters");
  if (r->struct_size != (int)sizeof(InfernoRope))
    return set_error(INFERNO_EINVAL, "rope: struct_size %d, expected %d", r->struct_size, (int)sizeof(InfernoRope));
  const int es = longctx_type_size(r->type);
  if (!es) return set_error(INFERNO_EINVAL, "rope: type %d is not F32, F16 or BF16", r->type);
  if (r->n_tokens < 0 || r->n_heads < 0 || r->n_kv_heads < 0 || r->head_dim < 1 || r->head_dim > 8192)
    return set_error(INFERNO_EINVAL, "rope: bad sizes (%d tokens, %d / %d heads of %d)", r->n_tokens, r->n_heads,
                     r->n_kv_heads, r->head_dim);
  if (r->rope_dim < 2 || r->rope_dim % 2 || r->rope_dim > r->head_dim || r->rope_dim > 2 * ROPE_MAX_PAIRS)
    return set_error(INFERNO_EINVAL, "rope: rope_dim %d is not even or outside 2..min(%d, %d)", r->rope_dim,
                     r->head_dim, 2 * ROPE_MAX_PAIRS);
  if (r->layout != INFERNO_ROPE_HALF && r->layout != INFERNO_ROPE_INTERLEAVED)
    return set_error(INFERNO_EINVAL, "rope: layout %d", r->layout);
  if (r->scaling < INFERNO_ROPE_SCALE_NONE || r->scaling > INFERNO_ROPE_SCALE_PARTS)
    return set_error(INFERNO_EINVAL, "rope: scaling %d", r->scaling);
  if (r->inverse != 0 && r->inverse != 1) return set_error(INFERNO_EINVAL, "rope: inverse %d", r->inverse);
  if (!(r->theta > 1.0f) || !std::isfinite(r->theta)) return set_error(INFERNO_EINVAL, "rope: theta %g", r->theta);
  if (r->scaling && (!(r->factor > 0.0f) || !std::isfinite(r->factor)))
    return set_error(INFERNO_EINVAL, "rope: factor %g", r->factor);
  const double fast = r->beta_fast == 0.0f ? 32.0 : r->beta_fast, slow = r->beta_slow == 0.0f ? 1.0 : r->beta_slow;
  if (r->scaling == INFERNO_ROPE_SCALE_PARTS &&
      (r->orig_ctx < 1 || !(fast > 0.0) || !(slow > 0.0) || !std::isfinite(fast) || !std::isfinite(slow)))
    return set_error(INFERNO_EINVAL, "rope: orig_ctx %d, beta_fast %g, beta_slow %g", r->orig_ctx, fast, slow);
  if (!(r->mscale >= 0.0f) || !std::isfinite(r->mscale)) return set_error(INFERNO_EINVAL, "rope: mscale %g", r->mscale);
  if (r->n_heads > 65536 || r->n_kv_heads > 65536) return set_error(INFERNO_EINVAL, "rope: too many heads");
  const bool has_q = r->n_heads > 0, has_k = r->n_kv_heads > 0 && r->k, has_v = r->v != nullptr;
  if (r->n_tokens == 0) return 0;
  if (!r->positions) return set_error(INFERNO_EINVAL, "rope: positions missing");
  if (has_q && (!r->q || !r->q_out)) return set_error(INFERNO_EINVAL, "rope: q or q_out missing");
  if (has_k && !r->k_out) return set_error(INFERNO_EINVAL, "rope: k_out missing");
  if (has_v && (!r->slots || !r->v_out || r->n_kv_heads < 1))
    return set_error(INFERNO_EINVAL, "rope: v needs slots, v_out and KV heads");
  if (r->slots && r->n_rows < 0) return set_error(INFERNO_EINVAL, "rope: n_rows %d", r->n_rows);
  if (!has_q && !has_k && !has_v) return 0;

  // rows, their overlaps and the widest common access
  const long long qw = (long long)r->n_heads * r->head_dim, kw = (long long)r->n_kv_heads * r->head_dim;
  const long long out_rows = r->slots ? r->n_rows : r->n_tokens;
  auto rows = [&](const void* p, long long stride, long long width, long long count) {
    return Rows{(const char*)p, stride * es, width * es, count};
  };
  const Rows in[3] = {rows(has_q ? r->q : nullptr, r->q_stride, qw, r->n_tokens),
                      rows(has_k ? r->k : nullptr, r->k_stride, kw, r->n_tokens),
                      rows(has_v ? r->v : nullptr, r->v_stride, kw, r->n_tokens)};
  const Rows out[3] = {rows(has_q ? r->q_out : nullptr, r->q_out_stride, qw, r->n_tokens),
                       rows(has_k ? r->k_out : nullptr, r->k_out_stride, kw, out_rows),
                       rows(has_v ? r->v_out : nullptr, r->v_out_stride, kw, out_rows)};
  static const char* const names[3] = {"q", "k", "v"};
  for (int i = 0; i < 3; ++i) {
    for (const Rows* a : {&in[i], &out[i]}) {
      if (!a->p) continue;
      if (a->stride < 0 || (a->count > 1 && a->stride < a->width))
        return set_error(INFERNO_EINVAL, "rope: a stride of %s is less than its row", names[i]);
      if (a->stride > (1ll << 50)) return set_error(INFERNO_EINVAL, "rope: a stride of %s is too large", names[i]);
      if ((uintptr_t)a->p % es) return set_error(INFERNO_EINVAL, "rope: %s is not aligned to its type", names[i]);
    }
    for (int j = 0; j < 3; ++j) {
      if (j > i && rows_overlap(out[i], out[j]))
        return set_error(INFERNO_EINVAL, "rope: %s_out overlaps %s_out", names[i], names[j]);
      const bool in_place = i == j && !(r->slots && i > 0) && out[i].p == in[j].p &&
                            (out[i].stride == in[j].stride || r->n_tokens == 1);
      if (!in_place && rows_overlap(out[i], in[j]))
        return set_error(INFERNO_EINVAL, "rope: %s_out overlaps %s", names[i], names[j]);
    }
  }
  int rc = longctx_check_device(out[0].p ? out[0].p : out[1].p ? out[1].p : out[2].p, "rope");
  if (rc) return rc;
  const bool ilv = r->layout == INFERNO_ROPE_INTERLEAVED;
  long long all = (long long)r->head_dim * es | (long long)r->rope_dim * es;
  if (!ilv) all |= (long long)r->rope_dim / 2 * es;
  for (int i = 0; i < 3; ++i)
    for (const Rows* a : {&in[i], &out[i]})
      if (a->p) all |= (long long)(uintptr_t)a->p | a->stride;
  int vec = 16 / es;
  while (vec > 1 && all % (vec * es)) vec /= 2;

  RopeParams p{};
  p.q = in[0].p, p.k = in[1].p, p.v = in[2].p;
  p.qo = (void*)out[0].p, p.ko = (void*)out[1].p, p.vo = (void*)out[2].p;
  p.qs = r->q_stride, p.ks = r->k_stride, p.vs = r->v_stride;
  p.qos = r->q_out_stride, p.kos = r->k_out_stride, p.vos = r->v_out_stride;
  p.positions = r->positions;
  p.slots = r->slots;
  p.freq_factors = r->freq_factors;
  p.n_tokens = r->n_tokens;
  p.n_rows = r->n_rows;
  p.head_dim = r->head_dim;
  p.rope_dim = r->rope_dim;
  const int half = r->rope_dim / 2;
  const int rv = ilv && vec < 2 ? 2 : vec;
  p.rot_items = (ilv ? r->rope_dim : half) / rv;
  const uint32_t per_head = p.rot_items + (r->head_dim - r->rope_dim) / vec;
  p.q_items = has_q ? r->n_heads * per_head : 0;
  p.k_items = p.q_items + (has_k ? r->n_kv_heads * per_head : 0);
  p.items = p.k_items + (has_v ? (uint32_t)(kw / vec) : 0);
  p.by_head = FastDiv(per_head);
  p.by_items = FastDiv(p.items);
  p.sign = r->inverse ? -1.0f : 1.0f;
  p.gain = r->mscale != 0.0f ? r->mscale
           : r->scaling == INFERNO_ROPE_SCALE_PARTS && r->factor > 1.0f ? (float)(0.1 * std::log((double)r->factor) + 1.0)
                                                                        : 1.0f;
  // f_i by repeated multiplication: 256 steps lose at most 2^-44 of f_i
  const double two_pi = 6.283185307179586476925286766559;
  const double ratio = std::pow((double)r->theta, -2.0 / r->rope_dim);
  double low = 0, high = 0;
  if (r->scaling == INFERNO_ROPE_SCALE_PARTS) {
    auto dim = [&](double turns) {
      return r->rope_dim * std::log(r->orig_ctx / (two_pi * turns)) / (2.0 * std::log((double)r->theta));
    };
    low = std::max(std::floor(dim(fast)), 0.0);
    high = std::min(std::ceil(dim(slow)), r->rope_dim - 1.0);
  }
  double f = 1.0 / two_pi;
  for (int i = 0; i < half; ++i, f *= ratio) {
    double g = f;
    if (r->scaling == INFERNO_ROPE_SCALE_LINEAR) g = f / r->factor;
    if (r->scaling == INFERNO_ROPE_SCALE_PARTS) {
      const double ramp = std::min(std::max((i - low) / std::max(high - low, 0.001), 0.0), 1.0);
      g = f * (1.0 - ramp) + f / r->factor * ramp;
    }
    p.turns[i] = g;
  }

  // tokens per block: enough that every thread has an angle to compute, fewer
  // when there are too few tokens to fill the SMs; then slices of about eight
  // items per thread, down to one per thread when there are few
  int dev = 0;
  INF_CUDA_TRY(cudaGetDevice(&dev));
  const long long sms = num_sms(dev);
  long long tb = std::max(1, ROPE_THREADS / half);
  tb = std::max(1ll, std::min(tb, r->n_tokens / (2 * sms)));
  while (tb > 1 && tb * p.items > (1ll << 30)) tb /= 2;
  p.tb = (int)tb;
  const long long blocks = (r->n_tokens + tb - 1) / tb;
  const long long per_block = tb * p.items;
  long long per_thread = std::min(8ll, std::max(1ll, blocks * per_block / (2 * sms * ROPE_THREADS)));
  long long slices = (per_block + per_thread * ROPE_THREADS - 1) / (per_thread * ROPE_THREADS);
  slices = std::min(slices, 65535ll);
  p.slice = (uint32_t)((per_block + slices - 1) / slices);
  const dim3 grid((unsigned)blocks, (unsigned)slices);
  const size_t smem = (size_t)tb * half * sizeof(float2);
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = r->type == INFERNO_F32   ? rope_launch<float>(p, vec, ilv, grid, smem, st)
                        : r->type == INFERNO_F16 ? rope_launch<__half>(p, vec, ilv, grid, smem, st)
                                                 : rope_launch<__nv_bfloat16>(p, vec, ilv, grid, smem, st);
  return e == cudaSuccess ? 0 : set_error(INFERNO_ECUDA, "rope launch: %s", cudaGetErrorString(e));
}
