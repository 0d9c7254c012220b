// Rotary positions of q and k with the append of k and v to cache rows
// (inferno_rope).
//
// A pair (a, b) of a head becomes (a cos - b sin, a sin + b cos) with the angle
// positions[t] * f_i.  A block takes a few tokens: its threads first put cos and
// sin of the tokens' angles into shared memory, once for all heads.  Then a team
// of threads, one per 16-byte column of a head (a column of the half layout is two
// vectors, rope_dim / 2 apart), takes four heads (or two) of a token at a time: cos and
// sin of a column are read once for them, and the loads of all are in flight together.
// (One vector per thread and index computation was bound by instructions: 96 us for
// 16383 tokens x 40 heads of 128 bf16, and more items in flight only made it slower.)
//
// Angles: f_i / (2 pi), the turns per position, is a 64-bit fraction, so its product
// with the position modulo 2^64 is the fraction of a turn that is left, whole turns
// dropped; that goes to sincospi in fp32.  The frequency is off by 2^-54 of itself (see
// the host) and 2^-64, so up to position 2^31 - 1 (2^28.4 turns) the angle is off by
// 2 pi (2^-26 + 2^-26), 2e-7, from it and from the rounding to fp32; by half of that up
// to position 2^28.  With freq_factors the frequency, in 64 bits of a unit of its own, is
// taken apart into a double and its rest, divided by the factor and multiplied exactly.
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

struct RopeParams {
  const void *q, *k, *v;
  void *qo, *ko, *vo;
  long long qs, ks, vs, qos, kos, vos;   // elements between token rows
  const int *positions, *slots;
  const float* freq_factors;
  int n_tokens, n_heads, n_kv, n_rows, head_dim, rope_dim;
  int tb;                                // tokens per block
  int cols, rot_cols;                    // columns of a head; those that are rotated
  int teams;                             // teams of a block (cols threads each, at most a block)
  uint32_t q_units, units;               // units (a few heads of one token): of q, of q and k
  uint32_t slice;                        // units of one block (over its tb tokens)
  uint32_t v_cols;                       // vectors of a v row (0: none)
  uint32_t v_slice;                      // v vectors of one block (over its tb tokens)
  FastDiv by_units, by_v;
  float gain, sign;                      // factor of cos and sin; -1: rotate back
  // f_i / (2 pi) times 2^64, modulo 2^64; with freq_factors not divided by them, and not
  // modulo 2^64 but in `unit`
  unsigned long long turns[ROPE_MAX_PAIRS];
  double unit;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T x[V];
};

// V elements <-> fp32, 16-bit types two at a time where there are two
template <typename T, int V>
__device__ __forceinline__ void unpack(const Vec<T, V>& v, float (&f)[V]) {
  if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = v.x[i];
  } else if constexpr (V == 1) {
    f[0] = (float)v.x[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      float2 y;
      if constexpr (std::is_same_v<T, __half>) y = __half22float2(*(const __half2*)&v.x[i]);
      else y = __bfloat1622float2(*(const __nv_bfloat162*)&v.x[i]);
      f[i] = y.x, f[i + 1] = y.y;
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> pack(const float (&f)[V]) {
  Vec<T, V> v;
  if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int i = 0; i < V; ++i) v.x[i] = f[i];
  } else if constexpr (V == 1) {
    v.x[0] = (T)f[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      if constexpr (std::is_same_v<T, __half>) *(__half2*)&v.x[i] = __floats2half2_rn(f[i], f[i + 1]);
      else *(__nv_bfloat162*)&v.x[i] = __floats2bfloat162_rn(f[i], f[i + 1]);
    }
  }
  return v;
}

// Heads of a unit: four, but two where a column is two vectors of eight values,
// whose 64 fp32 values of four heads leave too few registers for four blocks per
// SM (16383 tokens x 40 heads of 128 bf16: 95 us with four, 74 us with two)
template <typename T, int V, bool ILV>
__host__ __device__ constexpr int rope_heads() {
  return V == 8 && !ILV ? 2 : 4;
}

// half turns, less whole turns, of a pair with a factor w at a position
__device__ __forceinline__ float rope_half_turns(unsigned long long turns, double unit, double w, double at) {
  const double f = (double)(turns & ~0x7ffull) * unit, f_rest = (double)(turns & 0x7ffull) * unit;
  const double inv = 1.0 / w, g = f * inv;
  const double rest = g == 0.0 ? 0.0 : (fma(-g, w, f) + f_rest) * inv;       // 0: an infinite factor
  const double turn = g * at;
  return 2.0f * (float)(turn - rint(turn) + (fma(g, at, -turn) + rest * at));
}

// V: elements of one access (the widest that sizes, strides and pointers
// allow).  ILV: interleaved pairs; a column then holds whole pairs.
template <typename T, int V, bool ILV>
__global__ void __launch_bounds__(ROPE_THREADS, 4) rope_kernel(const __grid_constant__ RopeParams p) {
  extern __shared__ float2 cs[];                     // [tb][rope_dim / 2] (cos, sin)
  using Vt = Vec<T, V>;
  constexpr bool TWO = !ILV || V == 1;               // a column is two vectors
  constexpr int NP = ILV ? (V == 1 ? 1 : V / 2) : V; // pairs of one rotated column
  constexpr int HB = rope_heads<T, V, ILV>();        // heads of a unit
  const int half = p.rope_dim >> 1;
  const int t0 = blockIdx.x * p.tb, nt = min(p.tb, p.n_tokens - t0);
  for (int i = threadIdx.x; i < nt * half; i += ROPE_THREADS) {
    const int t = i / half, c = i - t * half;
    const int pos = __ldg(p.positions + t0 + t);
    // as a double it is one load of a constant, whose lanes differ and go one by one; as
    // an integer two, and every call 0.15 us longer
    const unsigned long long turns = __double_as_longlong(((const double*)p.turns)[c]);
    float half_turns;
    if (!p.freq_factors) {
      const unsigned long long left = turns * (unsigned long long)(long long)pos + 0x80000000ull;
      half_turns = (float)(int)(left >> 32) * 0x1p-31f;            // rounded to 2^-32 turns
    } else {
      half_turns = rope_half_turns(turns, p.unit, __ldg(p.freq_factors + c), pos);
    }
    float sn, cn;
    sincospif(half_turns, &sn, &cn);
    cs[i] = make_float2(cn * p.gain, sn * p.gain * p.sign);
  }
  __syncthreads();

  // ---- q and k ----
  const int width = min(p.cols, ROPE_THREADS), team = threadIdx.x / width, col0 = threadIdx.x - team * width;
  const uint32_t end = min((blockIdx.y + 1) * p.slice, (uint32_t)nt * p.units);
  if (team < p.teams) {
    for (uint32_t unit = blockIdx.y * p.slice + team; unit < end; unit += p.teams) {
      const uint32_t tl = p.by_units.div(unit), u = unit - tl * p.units;
      const int t = t0 + (int)tl;
      const bool isq = u < p.q_units;
      const int h0 = (int)(isq ? u : u - p.q_units) * HB, nh = min(HB, (isq ? p.n_heads : p.n_kv) - h0);
      long long row = t;
      if (!isq && p.slots) {
        row = __ldg(p.slots + t);
        if (row < 0 || row >= p.n_rows) continue;
      }
      const T* src0 = (isq ? (const T*)p.q + (long long)t * p.qs : (const T*)p.k + (long long)t * p.ks) + (long long)h0 * p.head_dim;
      T* dst0 = (isq ? (T*)p.qo + row * p.qos : (T*)p.ko + row * p.kos) + (long long)h0 * p.head_dim;
      for (int col = col0; col < p.cols; col += width) {
        const bool rot = col < p.rot_cols;
        const int off = !rot ? p.rope_dim + (col - p.rot_cols) * V : ILV ? 2 * NP * col : V * col;
        const int second = ILV ? 1 : half;           // from a vector to its partner
        const T* src = src0 + off;
        T* dst = dst0 + off;
        Vt a[HB], b[HB];
#pragma unroll
        for (int i = 0; i < HB; ++i)
          if (i < nh) {
            a[i] = *(const Vt*)(src + i * p.head_dim);
            if (TWO && rot) b[i] = *(const Vt*)(src + i * p.head_dim + second);
          }
        if (!rot) {
#pragma unroll
          for (int i = 0; i < HB; ++i)
            if (i < nh) *(Vt*)(dst + i * p.head_dim) = a[i];
          continue;
        }
        float2 w[NP];
#pragma unroll
        for (int i = 0; i < NP; ++i) w[i] = cs[tl * half + col * NP + i];
#pragma unroll
        for (int i = 0; i < HB; ++i)
          if (i < nh) {
            float x[V], y[V];
            unpack<T, V>(a[i], x);
            if constexpr (TWO) {
              unpack<T, V>(b[i], y);
#pragma unroll
              for (int j = 0; j < V; ++j) {
                const float xr = x[j] * w[j].x - y[j] * w[j].y;
                y[j] = x[j] * w[j].y + y[j] * w[j].x;
                x[j] = xr;
              }
              *(Vt*)(dst + i * p.head_dim + second) = pack<T, V>(y);
            } else {
#pragma unroll
              for (int j = 0; j < NP; ++j) {
                const float xr = x[2 * j] * w[j].x - x[2 * j + 1] * w[j].y;
                x[2 * j + 1] = x[2 * j] * w[j].y + x[2 * j + 1] * w[j].x;
                x[2 * j] = xr;
              }
            }
            *(Vt*)(dst + i * p.head_dim) = pack<T, V>(x);
          }
      }
    }
  }

  // ---- v: copied ----
  if (!p.v_cols) return;
  const uint32_t v_end = min((blockIdx.y + 1) * p.v_slice, (uint32_t)nt * p.v_cols);
  for (uint32_t e0 = blockIdx.y * p.v_slice + threadIdx.x; e0 < v_end; e0 += HB * ROPE_THREADS) {
    Vt x[HB];
    T* dst[HB];
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      dst[i] = nullptr;
      const uint32_t e = e0 + i * ROPE_THREADS;
      if (e >= v_end) continue;
      const uint32_t tl = p.by_v.div(e), c = e - tl * p.v_cols;
      const int t = t0 + (int)tl;
      const long long row = __ldg(p.slots + t);
      if (row < 0 || row >= p.n_rows) continue;
      dst[i] = (T*)p.vo + row * p.vos + (long long)c * V;
      x[i] = *(const Vt*)((const T*)p.v + (long long)t * p.vs + (long long)c * V);
    }
#pragma unroll
    for (int i = 0; i < HB; ++i)
      if (dst[i]) *(Vt*)dst[i] = x[i];
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
  if (r->struct_size && r->struct_size != (int)sizeof(InfernoRope))
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
  if (((uintptr_t)r->positions | (uintptr_t)r->slots | (uintptr_t)r->freq_factors) % 4)
    return set_error(INFERNO_EINVAL, "rope: positions, slots or freq_factors is not aligned to 4 bytes");
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
  int rc = longctx_check_device({in[0].p, in[1].p, in[2].p, out[0].p, out[1].p, out[2].p, r->positions, r->slots, r->freq_factors}, "rope");
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
  p.n_heads = has_q ? r->n_heads : 0;
  p.n_kv = has_k ? r->n_kv_heads : 0;
  p.n_rows = r->n_rows;
  p.head_dim = r->head_dim;
  p.rope_dim = r->rope_dim;
  const int half = r->rope_dim / 2;
  p.rot_cols = ilv ? r->rope_dim / std::max(vec, 2) : half / vec;
  p.cols = p.rot_cols + (r->head_dim - r->rope_dim) / vec;
  p.teams = std::max(1, ROPE_THREADS / p.cols);
  const int hb = vec == 8 && !ilv ? rope_heads<__half, 8, false>() : rope_heads<float, 4, false>();
  p.q_units = (p.n_heads + hb - 1) / hb;
  p.units = p.q_units + (p.n_kv + hb - 1) / hb;
  p.v_cols = has_v ? (uint32_t)(kw / vec) : 0;
  p.by_units = FastDiv(std::max(1u, p.units));
  p.by_v = FastDiv(std::max(1u, p.v_cols));
  p.sign = r->inverse ? -1.0f : 1.0f;
  p.gain = r->mscale != 0.0f ? r->mscale
           : r->scaling == INFERNO_ROPE_SCALE_PARTS && r->factor > 1.0f ? (float)(0.1 * std::log((double)r->factor) + 1.0)
                                                                        : 1.0f;
  // f_i by repeated multiplication in extended precision (64 bits): the ratio is off by
  // 2^-63 of itself and each product by 2^-64, so 255 steps lose 2^-54 of f_i.  (In
  // double they lost 1e-6 in the angle at far positions, or 2e-5 with theta 1.5, whose
  // later pairs turn nearly as fast as the first.)  The ratio is pow's in double after
  // one Newton step for theta ratio^half = 1: powl takes 400 ns of a call of 4 us.
  const double two_pi = 6.283185307179586476925286766559;
  long double ratio = std::pow((double)r->theta, -2.0 / r->rope_dim), power = r->theta, square = ratio;
  for (int n = half; n; n >>= 1, square *= square)
    if (n & 1) power *= square;
  ratio -= ratio * (power - 1.0L) / half;
  double low = 0, high = 0;
  if (r->scaling == INFERNO_ROPE_SCALE_PARTS) {
    auto dim = [&](double turns) {
      return r->rope_dim * std::log(r->orig_ctx / (two_pi * turns)) / (2.0 * std::log((double)r->theta));
    };
    low = std::max(std::floor(dim(fast)), 0.0);
    high = std::min(std::ceil(dim(slow)), r->rope_dim - 1.0);
  }
  long double f = 1.0L / 6.283185307179586476925286766559005768L;
  // 64 bits of the largest, which is not the first pair's where parts are made faster
  int unit_exp;
  std::frexp(r->scaling == INFERNO_ROPE_SCALE_LINEAR || (r->scaling == INFERNO_ROPE_SCALE_PARTS && r->factor < 1.0f) ? f / r->factor : f,
             &unit_exp);
  p.unit = std::ldexp(1.0, unit_exp - 64);
  for (int i = 0; i < half; ++i, f *= ratio) {
    long double g = f;
    if (r->scaling == INFERNO_ROPE_SCALE_LINEAR) g = f / r->factor;
    if (r->scaling == INFERNO_ROPE_SCALE_PARTS) {
      const long double ramp = std::min(std::max((i - low) / std::max(high - low, 0.001), 0.0), 1.0);
      g = f * (1.0L - ramp) + f / r->factor * ramp;
    }
    if (p.freq_factors) {
      p.turns[i] = (unsigned long long)(g / p.unit);
    } else {
      p.turns[i] = (unsigned long long)((g < 1.0L ? g : g - std::floor(g)) * 0x1p64L);
    }
  }

  // tokens per block: about four units for every team, fewer when there are too
  // few tokens to give every SM two blocks; then the units of a block are cut into
  // slices (which compute the angles again) until there are
  int dev = 0;
  INF_CUDA_TRY(cudaGetDevice(&dev));
  const long long sms = num_sms(dev);
  const long long work = std::max<long long>(p.units, (p.v_cols + (long long)hb * p.cols - 1) / ((long long)hb * p.cols));
  long long tb = 1;
  while (tb < 16 && tb * work < 4ll * p.teams && tb * 2 * half <= 1024) tb *= 2;
  while (tb > 1 && (r->n_tokens + tb - 1) / tb < 2 * sms) tb /= 2;
  p.tb = (int)tb;
  const long long blocks = (r->n_tokens + tb - 1) / tb;
  long long slices = std::max(1ll, std::min((2 * sms + blocks - 1) / blocks, (tb * work + p.teams - 1) / p.teams));
  slices = std::max(slices, (tb * work + 64ll * p.teams - 1) / (64ll * p.teams));
  slices = std::min(slices, 65535ll);
  p.slice = (uint32_t)((tb * p.units + slices - 1) / slices);
  p.v_slice = (uint32_t)((tb * p.v_cols + slices - 1) / slices);
  const dim3 grid((unsigned)blocks, (unsigned)slices);
  const size_t smem = (size_t)tb * half * sizeof(float2);
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = r->type == INFERNO_F32   ? rope_launch<float>(p, vec, ilv, grid, smem, st)
                        : r->type == INFERNO_F16 ? rope_launch<__half>(p, vec, ilv, grid, smem, st)
                                                 : rope_launch<__nv_bfloat16>(p, vec, ilv, grid, smem, st);
  return e == cudaSuccess ? 0 : set_error(INFERNO_ECUDA, "rope launch: %s", cudaGetErrorString(e));
}
