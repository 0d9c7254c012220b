// The shared-prefix part of inferno_attention_cached for 16-bit types and many
// query rows: all tokens of all sequences attend to the same keys, so a KV head's
// rows form the 128-row operand of tcgen05 and K / V are read once per 128 rows.
//
// A CTA takes 128 query rows of one KV head against one split of the prefix, in
// tiles of 64 keys:
//   S = Q K^T   A = Q tile, B = K tile in shared memory, S in TMEM (two buffers)
//   P = exp2(scale S - r), rounded to the 16-bit type (half a step of each weight, as
//   in attn_cached.cu; the sum takes it unrounded), back into S's columns
//   O += P V    A = P in TMEM, B = V tile, N-major as it lies in the cache
// Warps 0-3: softmax, one thread per row (TMEM lane); r, the reference of a row, follows
// its running maximum, and O is rescaled, only when that outgrows it by 2^8 (fp16 2^4),
// since P and the sums hold that much headroom.  Warp 4: K and V tiles by TMA.  Warp 5: issues the
// MMAs; S of the next tile is issued before P V of this one.  Two CTAs per SM (one at
// head_dim 256) fill each other's gaps.
//
// Bound: bytes of K and V up to 128 rows per KV head (a 64-key tile of head_dim 128
// takes 1460 clocks of an SM's share of HBM, about 640 of the tensor pipe and 512
// of the exponential unit); above that the exponentials and MMAs.
#include <algorithm>
#include <mutex>
#include <type_traits>
#include <cuda_bf16.h>
#include "internal.h"
#include "tc.cuh"
#include "attn_cached.h"
#include "longctx.h"
#include "../../include/inferno_b200.h"

namespace inf {

__device__ int ap_error;            // first bounded wait that ran out (DevErr)

namespace {

constexpr int AP_M = 128, AP_N = 64;
constexpr int AP_THREADS = 192;

// P_EXP: log2 of P at the maximum when the reference was set (ac_ref); sum and O are
// scaled alike.  SLACK: log2 of what P may exceed that by before the reference is
// raised.  fp16 has its full precision down to 2^-14 only, and nothing below 2^-25:
// 2^11 at the maximum and 2^15 at most leave it down to 2^-25 (and something down to
// 2^-36) of the maximum.
template <typename T>
struct ApType { static constexpr int P_EXP = 0; static constexpr float SLACK = 8.f; };
template <>
struct ApType<__half> { static constexpr int P_EXP = 11; static constexpr float SLACK = 4.f; };

template <int HD>
struct ApGeo {
  static constexpr int SUB = HD / 64;                        // 64-dim sub-tiles (128-byte rows)
  static constexpr int QBYTES = SUB * AP_M * 128;
  static constexpr int TILE = SUB * AP_N * 128;              // one K or V tile
  static constexpr int STAGES = HD == 64 ? 4 : 2;            // of K, and of V
  static constexpr int SMEM = 1024 + QBYTES + 2 * STAGES * TILE + 256;
  static constexpr int TMEM = HD == 256 ? 512 : 256;         // two S buffers and O
  static constexpr int CTAS = HD == 256 ? 1 : 2;
};

// A poll sleeps for up to about 4 us, so AP_POLLS give up after about two seconds.
// A CTA that gives up still waits for its own copies and MMAs in flight, and leaves
// NaN as the sums of its rows, so that what they join does not look like a result.
constexpr uint32_t AP_POLLS = 1u << 19;
__device__ __forceinline__ bool ap_wait(uint64_t* bar, uint32_t parity, uint32_t polls) {
  for (uint32_t i = 0; i < polls; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  atomicExch(&ap_error, DERR_MBAR_TIMEOUT);
  return false;
}
// D (+)= A[tmem] B[smem]
__device__ __forceinline__ void umma_ts_f16(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}
// Shared-memory descriptor of a SWIZZLE_128B operand whose rows run along its
// N (or M) extent: 64 elements of N per 128-byte row, eight rows of K per
// 1024-byte atom (stride byte offset), the next 64 of N `lbo` bytes on (leading
// byte offset).
__device__ __forceinline__ uint64_t ap_desc_n_major(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tmem_ld_x32(uint32_t a, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a)
      : "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t a, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(a),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t ap_pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&h;
  }
}

// row r of a KV head's rows -> token row (b * n_tok + t) and query head
__device__ __forceinline__ void ap_row(const AcParams& p, int kvh, int r, int& tok, int& h) {
  const int b = (int)p.by_seq.div(r), tg = r - b * (int)p.by_seq.d, t = (int)p.by_group.div(tg);
  tok = b * p.n_tok + t;
  h = kvh * p.group + tg - t * p.group;
}

struct alignas(64) ApMaps {
  CUtensorMap k, v;
};

template <typename T, int HD>
__global__ void __launch_bounds__(AP_THREADS, ApGeo<HD>::CTAS) ap_kernel(const __grid_constant__ AcParams p, const __grid_constant__ ApMaps maps, int row_tiles, uint32_t polls) {
  using G = ApGeo<HD>;
  constexpr int ST = G::STAGES;
  extern __shared__ uint8_t ap_smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_trigger();
  uint8_t* base = (uint8_t*)(((uintptr_t)ap_smem + 1023) & ~(uintptr_t)1023);
  uint8_t* s_q = base;                                  // [SUB][128 rows][128 B]
  uint8_t* s_k = s_q + G::QBYTES;                       // [ST][SUB][64 rows][128 B]
  uint8_t* s_v = s_k + ST * G::TILE;
  uint64_t* bars = (uint64_t*)(s_v + ST * G::TILE);
  uint64_t* k_full = bars;                // ST each
  uint64_t* k_empty = k_full + ST;
  uint64_t* v_full = k_empty + ST;
  uint64_t* v_empty = v_full + ST;
  uint64_t* s_full = v_empty + ST;        // 2
  uint64_t* p_full = s_full + 2;          // 2
  uint64_t* pv_done = p_full + 2;         // 1: phase j is P V of tile j
  uint64_t* o_done = pv_done + 1;         // 1: all of them
  uint64_t* drained = o_done + 1;         // 1: those issued before a wait ran out
  uint64_t* q_full = drained + 1;         // 1
  uint32_t* s_tmem = (uint32_t*)(q_full + 1);

  int x = blockIdx.x;
  const int split = x % p.p_splits;
  x /= p.p_splits;
  const int row0 = (x % row_tiles) * AP_M, kvh = x / row_tiles;
  const int nrows = p.batch * p.n_tok * p.group;
  const int j0 = split * p.p_split_len, j1 = min(p.prefix_len, j0 + p.p_split_len);
  const int tiles = (j1 - j0 + AP_N - 1) / AP_N;        // at least one

  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], AP_M);
    }
    mbar_init(pv_done, 1);
    mbar_init(o_done, 1);
    mbar_init(drained, 1);
    mbar_init(q_full, AP_M);
    fence_mbar_init();
  }
  if (warp == 5) {
    tmem_alloc(s_tmem, G::TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *s_tmem;
  const uint32_t t_o = tbase + 2 * AP_N;                // O behind the two S buffers

  if (warp == 4) {
    // ================= K / V producer =================
    if (lane == 0) {
      int k_issued = 0, v_issued = 0;
      for (int j = 0; j < tiles; ++j) {
        const int st = j % ST, key = j0 + j * AP_N;
        if (j >= ST && !ap_wait(&k_empty[st], ((j / ST) - 1) & 1, polls)) break;
        mbar_arrive_expect_tx(&k_full[st], G::TILE);
#pragma unroll
        for (int s = 0; s < G::SUB; ++s)
          tma_load_2d(s_k + st * G::TILE + s * AP_N * 128, &maps.k, kvh * HD + s * 64, key, &k_full[st]);
        k_issued = j + 1;
        if (j >= ST && !ap_wait(&v_empty[st], ((j / ST) - 1) & 1, polls)) break;
        mbar_arrive_expect_tx(&v_full[st], G::TILE);
#pragma unroll
        for (int s = 0; s < G::SUB; ++s)
          tma_load_2d(s_v + st * G::TILE + s * AP_N * 128, &maps.v, kvh * HD + s * 64, key, &v_full[st]);
        v_issued = j + 1;
      }
      // its own copies land before the CTA leaves: the last one of each stage
      for (int j = max(0, k_issued - ST); j < k_issued; ++j) ap_wait(&k_full[j % ST], (j / ST) & 1, AP_POLLS);
      for (int j = max(0, v_issued - ST); j < v_issued; ++j) ap_wait(&v_full[j % ST], (j / ST) & 1, AP_POLLS);
    }
    __syncwarp();
  } else if (warp == 5) {
    // ================= MMA issuer =================
    if (lane == 0) {
      constexpr uint32_t FMT = std::is_same_v<T, __half> ? 0u : (1u << 7) | (1u << 10);    // A and B: fp16 / bf16
      constexpr uint32_t id_s = umma_idesc_f16(AP_M, AP_N) | FMT;
      constexpr uint32_t id_o = umma_idesc_f16(AP_M, HD) | FMT | (1u << 16);               // B is N-major
      auto issue_s = [&](int j) {
        const uint32_t kb = smem_u32(s_k + (j % ST) * G::TILE), qb = smem_u32(s_q);
#pragma unroll
        for (int s = 0; s < G::SUB; ++s)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(tbase + (j & 1) * AP_N, umma_desc_sw128(qb + s * AP_M * 128 + k * 32),
                     umma_desc_sw128(kb + s * AP_N * 128 + k * 32), id_s, (s | k) != 0);
        umma_commit(&s_full[j & 1]);
        umma_commit(&k_empty[j % ST]);
      };
      bool ok = ap_wait(q_full, 0, polls) && ap_wait(&k_full[0], 0, polls);
      if (ok) {
        tc_fence_after();
        issue_s(0);
      }
      for (int j = 0; j < tiles && ok; ++j) {
        if (j + 1 < tiles) {
          // S(j + 1) takes the columns of P(j - 1), which P V (j - 1) reads
          ok = (j == 0 || ap_wait(pv_done, (j - 1) & 1, polls)) && ap_wait(&k_full[(j + 1) % ST], ((j + 1) / ST) & 1, polls);
          if (!ok) break;
          tc_fence_after();
          issue_s(j + 1);
        }
        ok = ap_wait(&p_full[j & 1], (j >> 1) & 1, polls) && ap_wait(&v_full[j % ST], (j / ST) & 1, polls);
        if (!ok) break;
        tc_fence_after();
        const uint32_t vb = smem_u32(s_v + (j % ST) * G::TILE);
#pragma unroll
        for (int k = 0; k < AP_N / 16; ++k)
          umma_ts_f16(t_o, tbase + (j & 1) * AP_N + k * 8, ap_desc_n_major(vb + k * 16 * 128, AP_N * 128), id_o,
                      (j | k) != 0);
        umma_commit(pv_done);
        umma_commit(&v_empty[j % ST]);
      }
      umma_commit(ok ? o_done : drained);
      if (!ok) ap_wait(drained, 0, AP_POLLS);     // no MMA in flight when TMEM is freed
    }
    __syncwarp();
  } else {
    // ================= softmax: one row per thread =================
    // a thread's 16-byte column is the same in all its rows; all copies in flight
    constexpr int CH = HD / 8, STEP = AP_M / CH;
    const int c = tid % CH;
#pragma unroll 8
    for (int r = tid / CH; r < AP_M; r += STEP) {
      int tok, h;
      ap_row(p, kvh, min(row0 + r, nrows - 1), tok, h);
      const T* src = (const T*)p.q + (long long)tok * p.q_stride + (long long)h * HD + c * 8;
      cp_async16(smem_u32(s_q) + (c >> 3) * AP_M * 128 + sw128_off(r, c & 7), src, row0 + r < nrows);
    }
    cp_commit();
    cp_wait<0>();
    fence_proxy_async_smem();
    mbar_arrive(q_full);

    const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
    float ref = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < tiles; ++j) {
      ok = ap_wait(&s_full[j & 1], (j >> 1) & 1, polls);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t t_s = tbase + lane_base + (j & 1) * AP_N;
      uint32_t u0[32], u1[32];
      tmem_ld_x32(t_s, u0);
      tmem_ld_x32(t_s + 32, u1);
      tmem_wait_ld();
      const int live = j1 - (j0 + j * AP_N);            // keys of this tile
      if (live < AP_N) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          if (i >= live) u0[i] = 0xff800000u;
          if (i + 32 >= live) u1[i] = 0xff800000u;
        }
      }
      // the largest logit: of scale * s, so the smallest s for a negative scale
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (p.scale_log2 < 0.f) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          if (i < live) u0[i] ^= 0x80000000u;
          if (i + 32 < live) u1[i] ^= 0x80000000u;
        }
      }
      float sc = fabsf(p.scale_log2);
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        mx[0] = fmaxf(mx[0], __uint_as_float(u0[i]));
        mx[1] = fmaxf(mx[1], __uint_as_float(u0[i + 1]));
        mx[2] = fmaxf(mx[2], __uint_as_float(u1[i]));
        mx[3] = fmaxf(mx[3], __uint_as_float(u1[i + 1]));
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
      // one rounding of scale S - r below leaves half a step of a far logit in P: such
      // rows are scaled, and so rounded, first
      if (fabsf(top) >= AC_FAR) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          u0[i] = __float_as_uint(__uint_as_float(u0[i]) * sc);
          u1[i] = __float_as_uint(__uint_as_float(u1[i]) * sc);
        }
        sc = 1.f;
      }
      constexpr int PE = ApType<T>::P_EXP;
      const float room = (PE && fabsf(ref) < AC_FAR ? (float)PE : 0.f) + ApType<T>::SLACK;
      const bool raise = j == 0 || top - ref > room;
      if (j > 0 && __any_sync(0xffffffffu, raise)) {
        // O holds P V up to tile j - 1 once that is done (j - 2 was before S (j) was
        // issued); P V (j) waits for this thread
        ok = ap_wait(pv_done, (j - 1) & 1, polls);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const float f = raise ? ex2(ref - ac_ref<PE>(top)) : 1.0f;    // ref = -inf: nothing gathered yet, f = 0
        l *= f;
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          uint32_t o[32];
          tmem_ld_x32(t_o + lane_base + c, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
          tmem_st_x32(t_o + lane_base + c, o);
        }
        tmem_wait_st();
      }
      if (raise) ref = ac_ref<PE>(top);
      const float z = ref == -INFINITY ? 0.f : ref;
      float sum[2] = {0.f, 0.f};
      uint32_t pk[32];
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const float a = ex2(fmaf(__uint_as_float(u0[i]), sc, -z)), b = ex2(fmaf(__uint_as_float(u0[i + 1]), sc, -z));
        sum[0] += a;
        sum[1] += b;
        pk[i >> 1] = ap_pack2<T>(a, b);
      }
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const float a = ex2(fmaf(__uint_as_float(u1[i]), sc, -z)), b = ex2(fmaf(__uint_as_float(u1[i + 1]), sc, -z));
        sum[0] += a;
        sum[1] += b;
        pk[16 + (i >> 1)] = ap_pack2<T>(a, b);
      }
      l += sum[0] + sum[1];
      tmem_st_x32(t_s, pk);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[j & 1]);
    }
    // ---- partial result ----
    // its own barrier: pv_done may be one or two phases on by now, and a parity
    // tells a phase only from its neighbours
    ok = ok && ap_wait(o_done, 0, polls);
    if (__all_sync(0xffffffffu, ok)) {
      tc_fence_after();
      // O leaves by whole 128-byte lines: 32 columns of a warp's 32 rows turn through
      // shared memory (the K ring, idle now; 36 floats apart, so that neither side
      // of the turn has two lanes of a phase on one bank), eight lanes per row
      float* turn = (float*)s_k + warp * 32 * 36;
      long long at[8];                                  // this lane's rows lane / 8 + 4 i
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = row0 + warp * 32 + i * 4 + (lane >> 3);
        int tok, h;
        ap_row(p, kvh, r, tok, h);
        at[i] = r < nrows ? ((long long)tok * p.nh + h) * p.p_splits + split : -1;
      }
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        __syncwarp();
        tmem_ld_x32(t_o + lane_base + c, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; i += 4) *(uint4*)(turn + lane * 36 + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (at[i] >= 0)
            *(uint4*)(p.part_o + at[i] * HD + c + (lane & 7) * 4) = *(const uint4*)(turn + (i * 4 + (lane >> 3)) * 36 + (lane & 7) * 4);
      }
      const int r = row0 + tid;
      if (r < nrows) {
        int tok, h;
        ap_row(p, kvh, r, tok, h);
        p.part_ml[((long long)tok * p.nh + h) * p.p_splits + split] = make_float2(ref, l);
      }
    } else if (row0 + tid < nrows) {
      int tok, h;
      ap_row(p, kvh, row0 + tid, tok, h);
      p.part_ml[((long long)tok * p.nh + h) * p.p_splits + split] = make_float2(0.f, NAN);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tbase, G::TMEM);
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn ap_encode() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = (EncodeTiledFn)p;
  });
  return fn;
}

// [rows][width] of a 16-bit type, box of 64 x 64, SWIZZLE_128B, zeros past the end
int ap_map(CUtensorMap* m, int type, const void* base, long long width, int rows) {
  EncodeTiledFn fn = ap_encode();
  if (!fn) return set_error(INFERNO_ECUDA, "attention_cached: cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)width * 2};
  const cuuint32_t box[2] = {64, AP_N};
  const cuuint32_t one[2] = {1, 1};
  const CUresult r = fn(m, type == INFERNO_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                        (void*)base, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(INFERNO_ECUDA, "attention_cached: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return 0;
}

template <typename T, int HD>
cudaError_t ap_launch(const AcParams& p, const ApMaps& maps, int row_tiles, uint32_t polls, cudaStream_t st) {
  using G = ApGeo<HD>;
  static DeviceOnce once;
  const cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(ap_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM);
  });
  if (e != cudaSuccess) return e;
  const long long blocks = (long long)row_tiles * p.nkv * p.p_splits;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  ap_kernel<T, HD><<<(unsigned)blocks, AP_THREADS, G::SMEM, st>>>(p, maps, row_tiles, polls);
  return cudaGetLastError();
}
template <typename T>
cudaError_t ap_launch_hd(int hd, const AcParams& p, const ApMaps& maps, int row_tiles, uint32_t polls, cudaStream_t st) {
  return hd == 64    ? ap_launch<T, 64>(p, maps, row_tiles, polls, st)
         : hd == 128 ? ap_launch<T, 128>(p, maps, row_tiles, polls, st)
                     : ap_launch<T, 256>(p, maps, row_tiles, polls, st);
}

}  // namespace

int ap_rows() { return AP_M; }
int ap_ctas_per_sm(int hd) { return hd == 256 ? ApGeo<256>::CTAS : ApGeo<128>::CTAS; }

int launch_attn_prefix_tc(int type, int hd, const AcParams& p, int row_tiles, bool give_up, cudaStream_t st) {
  ApMaps maps;
  const long long width = (long long)p.nkv * hd;
  int rc = ap_map(&maps.k, type, p.pk, width, p.prefix_len);
  if (!rc) rc = ap_map(&maps.v, type, p.pv, width, p.prefix_len);
  if (rc) return rc;
  const uint32_t polls = give_up ? 0 : AP_POLLS;
  const cudaError_t e = type == INFERNO_F16 ? ap_launch_hd<__half>(hd, p, maps, row_tiles, polls, st)
                                            : ap_launch_hd<__nv_bfloat16>(hd, p, maps, row_tiles, polls, st);
  return e == cudaSuccess ? 0 : set_error(INFERNO_ECUDA, "attention_cached launch: %s", cudaGetErrorString(e));
}

int attn_prefix_device_error(int device, int clear) {
  int before = 0, v = 0;
  cudaError_t e = cudaGetDevice(&before);
  if (e == cudaSuccess) e = cudaSetDevice(device);
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, ap_error, sizeof v);
  const int zero = 0;
  if (e == cudaSuccess && clear && v) e = cudaMemcpyToSymbol(ap_error, &zero, sizeof zero);
  cudaSetDevice(before);
  return e == cudaSuccess ? v : 0;
}

}  // namespace inf
