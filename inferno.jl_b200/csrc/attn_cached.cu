// Attention of a few new tokens per sequence over a shared prefix and the
// sequence's own cache (inferno_attention_cached).
//
//   out = sum_j p_j v_j,  p = softmax_j(scale q . k_j) over prefix and own rows
//
// Bound: the bytes of K and V, read once, while a KV head has few query rows
// (n_tokens x group for its own rows, batch x n_tokens x group for the prefix).
//
// ac_part_kernel: a CTA takes 16 R query rows of one KV head (prefix: of all
// sequences; own part: of one) against a range of keys (attn_cached.h says how they
// are cut).  Its warps form NG
// key groups of R warps; each group walks its own tiles of 16 keys with a ring of
// cp.async slots (a K or a V tile per slot, rows past the end zero-filled), each
// warp holds 16 rows: S = Q K^T and O += P V by mma.sync with the running
// maximum and sum of the softmax in registers.  mma.sync because a tile of
// 16 rows cannot fill the 128-row tcgen05 instruction and the kernel is bound by
// bytes; fp32 operands are carried as tf32 pairs (hi, lo) in three products,
// about 21 significant bits.  The groups merge in shared memory.
// ac_vec_kernel: the same for fp32 and few query rows, on the CUDA cores, a lane
// holding some dims of the rows and of the keys (see there).
// ac_finish_kernel: joins the partial results of a row, and adds the weights of the own
// rows to `scores` from the logits that the first kernel left.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <cuda_bf16.h>
#include "internal.h"
#include "common.cuh"
#include "attn_cached.h"
#include "longctx.h"
#include "../../include/inferno_b200.h"

namespace inf {

namespace {

constexpr int AC_SMS = 148;                     // of a B200
constexpr int AC_KT = 16;                       // keys per tile
constexpr int AC_SMEM = 227 * 1024, AC_SMEM_HALF = 112 * 1024;
constexpr int AC_FIN_THREADS = 256;

// P_EXP: log2 of the largest P (ac_ref); sum and O are scaled alike.  fp16 has its full
// precision down to 2^-14 only, and nothing below 2^-25: with the largest weight at
// 2^15 that is 2^-29 and 2^-40 of it, so that a long tail of small weights is not lost.
template <typename T>
struct AcType;
template <>
struct AcType<float> { static constexpr bool F32 = true; static constexpr int P_EXP = 0; };
template <>
struct AcType<__half> { static constexpr bool F32 = false; static constexpr int P_EXP = 15; };
template <>
struct AcType<__nv_bfloat16> { static constexpr bool F32 = false; static constexpr int P_EXP = 0; };

// geometry of one instantiation
template <typename T, int HD, int R>
struct AcGeo {
  static constexpr int ROW = HD * (int)sizeof(T);              // bytes of a K / V row of one head
  static constexpr int ITEM = AC_KT * ROW;                     // bytes of a ring slot
  // Q in registers; of fp32 above head_dim 64 they are too few, it stays in shared memory
  static constexpr bool QS = AcType<T>::F32 && HD > 64;
  static constexpr int QBYTES = QS ? 16 * R * ROW : 0;
  // two CTAs of four warps per SM, so that one streams while the other starts or
  // merges; one CTA of up to eight warps where the half SM does not hold three
  // slots per group (fp32 at head_dim 256)
  static constexpr int ML = 8 * 16 * 8;
  static constexpr bool TWO = (4 / R) * 3 * ITEM + QBYTES + ML <= AC_SMEM_HALF &&
                              4 * 16 * HD * 4 + ML <= AC_SMEM_HALF;   // the merge buffer takes the place of Q and ring
  static constexpr int CTAS = TWO ? 2 : 1;
  static constexpr int ROOM = (TWO ? AC_SMEM_HALF : AC_SMEM) - ML - QBYTES;
  static constexpr int NG0 = (TWO ? 4 : 8) / R;
  static constexpr int NG = NG0 * 3 * ITEM <= ROOM ? NG0 : NG0 / 2;
  static constexpr int NW = NG * R;
  static constexpr int THREADS = NW * 32;
  static constexpr int MAXSLOTS = ROOM / (NG * ITEM);
  static constexpr int SLOTS = MAXSLOTS > 6 ? 6 : MAXSLOTS;
  static constexpr int RING = NG * SLOTS * ITEM;
  static constexpr int MERGE = NW * 16 * HD * 4;
  static constexpr int BODY = QBYTES + RING > MERGE ? QBYTES + RING : MERGE;
  static constexpr int SMEM = BODY + NW * 16 * 8;
  static_assert(SLOTS >= 3 && SMEM <= (TWO ? AC_SMEM_HALF : AC_SMEM), "shared memory");
};

__device__ __forceinline__ void ldsm_x4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ float4 lds_f4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo: hi rounded to tf32's 11 significant bits (half up in magnitude),
// lo the exact rest, of which the instruction reads the leading 11 bits
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&h;
  }
}

// address of the 16-byte chunk c of row r of a tile; the exclusive-or spreads the
// rows that one access touches over all banks
template <int ROW>
__device__ __forceinline__ uint32_t tile_addr(uint32_t base, int r, int c) {
  return base + r * ROW + ((c ^ (r & 7)) << 4);
}

// bit k: row k of a tile (AC_KT rows of V) holds an infinity or NaN.  A whole warp.
template <typename T, int ROW>
__device__ __forceinline__ uint32_t ac_bad_rows(uint32_t tile, int lane) {
  constexpr int CH = ROW / 16;
  uint32_t bad = 0;
  for (int id = lane; id < AC_KT * CH; id += 32) {
    const float4 f = lds_f4(tile + id * 16);        // swizzled within the row: any order does
    const uint32_t x[4] = {__float_as_uint(f.x), __float_as_uint(f.y), __float_as_uint(f.z), __float_as_uint(f.w)};
    bool is = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, float>) is |= (x[i] & 0x7f800000u) == 0x7f800000u;
      else if constexpr (std::is_same_v<T, __half>) is |= (x[i] & 0x7c00u) == 0x7c00u || (x[i] & 0x7c000000u) == 0x7c000000u;
      else is |= (x[i] & 0x7f80u) == 0x7f80u || (x[i] & 0x7f800000u) == 0x7f800000u;
    }
    if (is) bad |= 1u << (id / CH);
  }
  return __reduce_or_sync(0xffffffffu, bad);
}

// what a CTA works on
struct AcWork {
  const uint8_t *k, *v;      // first key row of the KV head
  long long entry;           // own part: entry of its first row
  int j0, j1;                // keys
  int row0, nrows;           // rows of this CTA among its part's; their number
  int b;                     // own part: the sequence (prefix: -1)
  int kvh, split;            // prefix: the split
  int len;                   // own part: lens[b]
};

// row `r` of a part (prefix: over all sequences) -> (b, t, h)
__device__ __forceinline__ void ac_row(const AcParams& p, const AcWork& w, int r, int& b, int& t, int& h) {
  b = w.b;
  if (b < 0) {
    b = (int)p.by_seq.div(r);
    r -= b * (int)p.by_seq.d;
  }
  t = (int)p.by_group.div(r);
  h = w.kvh * p.group + (r - t * p.group);
}

// factor of a part with statistics (largest logit, sum) in a row whose largest
// logit is M.  A part without keys has weight 0; one whose logits are all NaN
// also has no largest logit, but its sum is NaN, and so is its weight here.
__device__ __forceinline__ float ac_weight(float2 ml, float M) {
  return ml.x == -INFINITY && ml.y == 0.f ? 0.f : exp2f(ml.x - M);
}

// CTAs of a launch: the prefix part's (row tiles of p_tiles), then the own part's
struct AcGrid {
  int p_blocks, p_tiles;
};

__device__ __forceinline__ int ac_len(const AcParams& p, int b) { return max(0, min(p.lens[b], p.max_len)); }
__device__ __forceinline__ int ac_blocks(int len) { return (len + AC_BLOCK - 1) / AC_BLOCK; }

// where an own-part CTA stands in the line of blocks (fewer than 2^30)
struct AcCursor {
  int pos, end;              // next block, end of the share
  int before, b;             // blocks of the sequences before b
  int group, u;              // the CTA's group and its KV head and row tile
};

// the segment at the cursor (sequence cur.b with `len` keys, up to the end of the
// share), and the cursor past it
template <typename T, int HD>
__device__ __forceinline__ void ac_take(const AcParams& p, AcCursor& cur, AcWork& w, int len) {
  constexpr int ROW = HD * (int)sizeof(T);
  const int off = cur.pos - cur.before, n = min(ac_blocks(len) - off, cur.end - cur.pos);
  cur.pos += n;
  w.b = cur.b;
  w.kvh = cur.u / p.o_tiles;
  w.row0 = (cur.u - w.kvh * p.o_tiles) * p.o_rows;
  w.nrows = p.n_tok * p.group;
  w.len = len;
  w.j0 = off * AC_BLOCK;
  w.j1 = min(len, w.j0 + n * AC_BLOCK);
  w.split = 0;
  w.entry = p.own_base + ((long long)(cur.group + cur.b) * (p.nkv * p.o_tiles) + cur.u) * p.o_rows;
  const long long base = (long long)cur.b * p.seq_stride * (int)sizeof(T) + (long long)w.kvh * ROW;
  w.k = (const uint8_t*)p.kc + base;
  w.v = (const uint8_t*)p.vc + base;
}
// the next segment; j0 = j1 when the share is done.  One thread.
template <typename T, int HD>
__device__ void ac_next(const AcParams& p, AcCursor& cur, AcWork& w) {
  w.j0 = w.j1 = 0;
  if (cur.pos >= cur.end) return;
  int len = ac_len(p, cur.b);
  while (cur.pos >= cur.before + ac_blocks(len)) {
    cur.before += ac_blocks(len);
    len = ac_len(p, ++cur.b);
  }
  ac_take<T, HD>(p, cur, w, len);
}

// this CTA's first segment.  One warp; lane 0 leaves cursor and work.
template <typename T, int HD>
__device__ void ac_first(const AcParams& p, AcGrid gr, int rows_per_cta, AcCursor& cur, AcWork& w) {
  const int lane = threadIdx.x & 31;
  if ((int)blockIdx.x < gr.p_blocks) {
    if (lane == 0) {
      int x = blockIdx.x;
      w.split = x % p.p_splits;
      x /= p.p_splits;
      w.row0 = (x % gr.p_tiles) * rows_per_cta;
      w.kvh = x / gr.p_tiles;
      w.b = -1;
      w.nrows = p.batch * p.n_tok * p.group;
      w.len = p.prefix_len;
      w.j0 = w.split * p.p_split_len;
      w.j1 = min(w.len, w.j0 + p.p_split_len);
      w.entry = 0;
      w.k = (const uint8_t*)p.pk + (long long)w.kvh * HD * (int)sizeof(T);
      w.v = (const uint8_t*)p.pv + (long long)w.kvh * HD * (int)sizeof(T);
      cur.pos = cur.end = 0;
    }
    return;
  }
  const int c = blockIdx.x - gr.p_blocks, units = p.nkv * p.o_tiles, group = c / units;
  // lane l sums the blocks of `per` consecutive sequences
  const int per = (p.batch + 31) / 32, b_lo = min(p.batch, lane * per), b_hi = min(p.batch, b_lo + per);
  int mine = 0, len = 0;
#pragma unroll 4
  for (int b = b_lo; b < b_hi; ++b) {
    len = ac_len(p, b);
    mine += ac_blocks(len);
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  const int all = __shfl_sync(0xffffffffu, incl, 31);
  const int share = max(1u, p.by_groups.div((uint32_t)(all + p.o_groups - 1)));
  const int pos = group * share, end = min(all, pos + share);
  if (c == 0) {
    if (lane == 0) p.head[0] = share;
    int before = incl - mine;
    for (int b = b_lo; b < b_hi; ++b) {
      p.head[1 + b] = before;
      before += ac_blocks(ac_len(p, b));
    }
  }
  if (pos >= end) {
    if (lane == 0) w.j0 = w.j1 = 0;
    return;
  }
  // the lane whose sequences hold pos
  if (incl - mine <= pos && pos < incl) {
    cur.group = group;
    cur.u = c - group * units;
    cur.pos = pos;
    cur.end = end;
    cur.before = incl - mine;
    cur.b = b_lo;
    if (per == 1) ac_take<T, HD>(p, cur, w, len);
    else ac_next<T, HD>(p, cur, w);
  }
}

// entry of row r (of the CTA's rows_per_cta) of a piece of work
__device__ __forceinline__ long long ac_entry(const AcParams& p, const AcWork& w, int r) {
  if (w.b >= 0) return w.entry + r;
  int b, t, h;
  ac_row(p, w, w.row0 + r, b, t, h);
  return ((long long)(b * p.n_tok + t) * p.nh + h) * p.p_splits + w.split;
}

// fp32: the logits of rows r and r + 8 of a part with keys 2 t4, 2 t4 + 1 and 8 more of
// the tile at kt, in the accumulator layout, in place of those of s that are NaN
template <int HD>
__device__ __forceinline__ void ac_plain_logits(const AcParams& p, const AcWork& w, int r, uint32_t kt, int t4, float (&s)[2][4]) {
  const float* q[2] = {nullptr, nullptr};
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (r + 8 * i < w.nrows) {
      int b, t, h;
      ac_row(p, w, r + 8 * i, b, t, h);
      q[i] = (const float*)p.q + (long long)(b * p.n_tok + t) * p.q_stride + (long long)h * HD;
    }
  float e[2][4] = {};
#pragma unroll 1
  for (int c = 0; c < HD / 4; ++c) {
    float4 x[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = q[i] ? *(const float4*)(q[i] + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 k = lds_f4(tile_addr<HD * 4>(kt, 8 * n + 2 * t4 + j, c));
#pragma unroll
        for (int i = 0; i < 2; ++i)
          e[n][2 * i + j] = fmaf(x[i].w, k.w, fmaf(x[i].z, k.z, fmaf(x[i].y, k.y, fmaf(x[i].x, k.x, e[n][2 * i + j]))));
      }
  }
#pragma unroll
  for (int a = 0; a < 8; ++a)
    if (s[a >> 2][a & 3] != s[a >> 2][a & 3]) s[a >> 2][a & 3] = e[a >> 2][a & 3];
}

// one piece of work of a CTA, from its first copies to its partial results
template <typename T, int HD, int R>
__device__ __forceinline__ void ac_part_segment(const AcParams& p, const AcWork w, uint8_t* smem) {
  using G = AcGeo<T, HD, R>;
  constexpr bool F32 = AcType<T>::F32;
  constexpr int ROW = G::ROW, ITEM = G::ITEM, SLOTS = G::SLOTS, GT = R * 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int grp = warp / R, rt = warp - grp * R;       // key group, row tile of the warp
  const int gtid = tid - grp * GT;                     // thread within the group
  const long long key_stride = (long long)p.nkv * ROW;

  const uint32_t s_q = smem_u32(smem);                            // with QS: [16 R][HD]
  uint8_t* ring_p = smem + G::QBYTES;
  const uint32_t ring = smem_u32(ring_p) + grp * SLOTS * ITEM;
  float2* s_ml = (float2*)(smem + G::BODY);                      // [NW][16]

  // tiles of this group: grp, grp + NG, ...; item 2 i is K of its i-th tile, 2 i + 1 V
  const int ntiles = (w.j1 - w.j0 + AC_KT - 1) / AC_KT;
  const int my_tiles = ntiles > grp ? (ntiles - grp + G::NG - 1) / G::NG : 0;
  const int items = 2 * my_tiles;
  auto issue = [&](int item) {
    if (item < items) {
      const int key0 = w.j0 + (grp + (item >> 1) * G::NG) * AC_KT;
      const uint8_t* src = (item & 1) ? w.v : w.k;
      const uint32_t dst = ring + (item % SLOTS) * ITEM;
      constexpr int CH = ROW / 16;
#pragma unroll
      for (int i = 0; i < AC_KT * CH / GT; ++i) {
        const int id = i * GT + gtid, r = id / CH, c = id % CH;
        const bool ok = key0 + r < w.j1;
        cp_async16(tile_addr<ROW>(dst, r, c), src + (ok ? (long long)(key0 + r) * key_stride : 0) + c * 16, ok);
      }
    }
    cp_commit();
  };
  if constexpr (G::QS) {     // Q ahead of the ring, part of its first copy group
    constexpr int CH = ROW / 16;
#pragma unroll 4
    for (int id = tid; id < 16 * R * CH; id += G::THREADS) {
      const int r = id / CH, c = id % CH;
      int b, t, h;
      ac_row(p, w, min(w.row0 + r, w.nrows - 1), b, t, h);
      cp_async16(tile_addr<ROW>(s_q, r, c), (const float*)p.q + (long long)(b * p.n_tok + t) * p.q_stride + (long long)h * HD + 4 * c,
                 w.row0 + r < w.nrows);
    }
  }
#pragma unroll
  for (int i = 0; i < SLOTS - 1; ++i) issue(i);

  // ---- Q: A fragments in registers (fp32: the float4 of each 16-byte column that
  // S takes of the two rows), or in shared memory ----
  uint32_t qf[F32 ? 1 : HD / 16][4];
  float4 qr[F32 && !G::QS ? HD / 16 : 1][2];
  const int r_lo = w.row0 + rt * 16 + g, r_hi = r_lo + 8;         // the two rows of this thread
  int lim_lo = 0, lim_hi = 0;                                     // keys they see
  {
    int b, t, h;
    const T *q_lo = nullptr, *q_hi = nullptr;
    if (r_lo < w.nrows) {
      ac_row(p, w, r_lo, b, t, h);
      q_lo = (const T*)p.q + (long long)(b * p.n_tok + t) * p.q_stride + (long long)h * HD;
      lim_lo = w.b < 0 ? w.len : w.len - p.n_tok + 1 + t;
    }
    if (r_hi < w.nrows) {
      ac_row(p, w, r_hi, b, t, h);
      q_hi = (const T*)p.q + (long long)(b * p.n_tok + t) * p.q_stride + (long long)h * HD;
      lim_hi = w.b < 0 ? w.len : w.len - p.n_tok + 1 + t;
    }
    if constexpr (!F32) {
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        const int d = 16 * k + 2 * t4;
        qf[k][0] = q_lo ? *(const uint32_t*)(q_lo + d) : 0u;
        qf[k][1] = q_hi ? *(const uint32_t*)(q_hi + d) : 0u;
        qf[k][2] = q_lo ? *(const uint32_t*)(q_lo + d + 8) : 0u;
        qf[k][3] = q_hi ? *(const uint32_t*)(q_hi + d + 8) : 0u;
      }
    } else if constexpr (G::QS) {
      cp_wait<SLOTS - 2>();
      __syncthreads();
    } else {
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        const int d = 4 * (8 * (i >> 1) + 2 * t4 + (i & 1));
        qr[i][0] = q_lo ? *(const float4*)(q_lo + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        qr[i][1] = q_hi ? *(const float4*)(q_hi + d) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
  }
  float* lg_lo = nullptr;
  float* lg_hi = nullptr;
  if (p.scores && w.b >= 0) {
    int b, t, h;
    if (r_lo < w.nrows) {
      ac_row(p, w, r_lo, b, t, h);
      lg_lo = p.logits + ((long long)(b * p.n_tok + t) * p.nh + h) * p.logit_stride;
    }
    if (r_hi < w.nrows) {
      ac_row(p, w, r_hi, b, t, h);
      lg_hi = p.logits + ((long long)(b * p.n_tok + t) * p.nh + h) * p.logit_stride;
    }
  }

  float o[HD / 8][4];
#pragma unroll
  for (int i = 0; i < HD / 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
  float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;

  auto landed = [&]() {
    cp_wait<SLOTS - 2>();
    if constexpr (R == 1) __syncwarp();
    else named_bar_sync(1 + grp, GT);
  };

  const bool busy = w.row0 + rt * 16 < w.nrows;      // the warp has rows; else it only copies
  for (int i = 0; i < my_tiles; ++i) {
    const int key0 = w.j0 + (grp + i * G::NG) * AC_KT;
    // ---- S = Q K^T ----
    landed();
    issue(2 * i + SLOTS - 1);
    if (!busy) {
      landed();
      issue(2 * i + 1 + SLOTS - 1);
      continue;
    }
    const uint32_t kt = ring + ((2 * i) % SLOTS) * ITEM;
    float s[2][4];
    if constexpr (!F32) {
      float c[2][2][4];              // even and odd k steps apart: shorter dependence chains
#pragma unroll
      for (int a = 0; a < 16; ++a) c[a >> 3][(a >> 2) & 1][a & 3] = 0.f;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        uint32_t kb[4];
        ldsm_x4(tile_addr<ROW>(kt, (lane >> 4) * 8 + (lane & 7), 2 * k + ((lane >> 3) & 1)), kb);
        mma16<T>(c[k & 1][0], qf[k], kb[0], kb[1]);
        mma16<T>(c[k & 1][1], qf[k], kb[2], kb[3]);
      }
#pragma unroll
      for (int a = 0; a < 8; ++a) s[a >> 2][a & 3] = c[0][a >> 2][a & 3] + c[1][a >> 2][a & 3];
    } else {
      // The tensor core truncates when it adds to its accumulator, so a long chain
      // drifts by half a step of the sum per product.  Chains are kept to four
      // products and added up in fp32 (rounded): 1.6e-6 -> 5e-7 of the result.
      // Six accumulators take turns, so that none waits for its last product.
      float hl[2][4], lh[2][4];      // hi lo and lo hi: small, one chain each
#pragma unroll
      for (int a = 0; a < 8; ++a) s[a >> 2][a & 3] = hl[a >> 2][a & 3] = lh[a >> 2][a & 3] = 0.f;
#pragma unroll
      for (int cg = 0; cg < HD / 32; ++cg) {
        float c[2][4];
#pragma unroll
        for (int a = 0; a < 8; ++a) c[a >> 2][a & 3] = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // four consecutive dims per thread, used as the k indices t4 and t4 + 4
          // of two k steps, the same dims of Q and K
          const int ch = 8 * cg + 2 * t4 + e;
          float4 qa, qb;
          if constexpr (G::QS) {
            qa = lds_f4(tile_addr<ROW>(s_q, rt * 16 + g, ch));
            qb = lds_f4(tile_addr<ROW>(s_q, rt * 16 + g + 8, ch));
          } else {
            qa = qr[2 * cg + e][0], qb = qr[2 * cg + e][1];
          }
          const float4 k0 = lds_f4(tile_addr<ROW>(kt, g, ch));
          const float4 k1 = lds_f4(tile_addr<ROW>(kt, g + 8, ch));
          const float qv[2][4] = {{qa.x, qb.x, qa.y, qb.y}, {qa.z, qb.z, qa.w, qb.w}};
          const float kv[2][2][2] = {{{k0.x, k0.y}, {k1.x, k1.y}}, {{k0.z, k0.w}, {k1.z, k1.w}}};
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            uint32_t ah[4], al[4], bh[2][2], bl[2][2];
#pragma unroll
            for (int x = 0; x < 4; ++x) split_tf32(qv[st][x], ah[x], al[x]);
#pragma unroll
            for (int x = 0; x < 4; ++x) split_tf32(kv[st][x >> 1][x & 1], bh[x >> 1][x & 1], bl[x >> 1][x & 1]);
#pragma unroll
            for (int n = 0; n < 2; ++n) mma_tf32(c[n], ah, bh[n][0], bh[n][1]);
#pragma unroll
            for (int n = 0; n < 2; ++n) mma_tf32(hl[n], ah, bl[n][0], bl[n][1]);
#pragma unroll
            for (int n = 0; n < 2; ++n) mma_tf32(lh[n], al, bh[n][0], bh[n][1]);
          }
        }
#pragma unroll
        for (int a = 0; a < 8; ++a) s[a >> 2][a & 3] += c[a >> 2][a & 3];
      }
#pragma unroll
      for (int a = 0; a < 8; ++a) s[a >> 2][a & 3] += hl[a >> 2][a & 3] + lh[a >> 2][a & 3];
      // An infinity in Q or K has the rest inf - inf, and so NaN for the logit that
      // may be -inf: such logits are formed again from the values themselves.
      bool odd = false;
#pragma unroll
      for (int a = 0; a < 8; ++a) odd |= s[a >> 2][a & 3] != s[a >> 2][a & 3];
      if (__any_sync(0xffffffffu, odd)) ac_plain_logits<HD>(p, w, r_lo, kt, t4, s);
    }
    // ---- running softmax ----
    float mx_lo = -INFINITY, mx_hi = -INFINITY;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int key = key0 + 8 * n + 2 * t4 + x;
        const bool in = key < w.j1;
        s[n][x] = in && key < lim_lo ? s[n][x] * p.scale_log2 : -INFINITY;
        s[n][2 + x] = in && key < lim_hi ? s[n][2 + x] * p.scale_log2 : -INFINITY;
        mx_lo = fmaxf(mx_lo, s[n][x]);
        mx_hi = fmaxf(mx_hi, s[n][2 + x]);
      }
#pragma unroll
    for (int of = 1; of <= 2; of <<= 1) {
      mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, of));
      mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, of));
    }
    if (lg_lo) {
#pragma unroll
      for (int n = 0; n < 2; ++n) *(float2*)(lg_lo + key0 + 8 * n + 2 * t4) = make_float2(s[n][0], s[n][1]);
    }
    if (lg_hi) {
#pragma unroll
      for (int n = 0; n < 2; ++n) *(float2*)(lg_hi + key0 + 8 * n + 2 * t4) = make_float2(s[n][2], s[n][3]);
    }
    constexpr int PE = AcType<T>::P_EXP;
    if (__any_sync(0xffffffffu, mx_lo > m_lo || mx_hi > m_hi)) {
      const float n_lo = fmaxf(m_lo, mx_lo), n_hi = fmaxf(m_hi, mx_hi);
      const float f_lo = n_lo == -INFINITY ? 1.f : exp2f(ac_ref<PE>(m_lo) - ac_ref<PE>(n_lo));
      const float f_hi = n_hi == -INFINITY ? 1.f : exp2f(ac_ref<PE>(m_hi) - ac_ref<PE>(n_hi));
      m_lo = n_lo, m_hi = n_hi;
      l_lo *= f_lo, l_hi *= f_hi;
#pragma unroll
      for (int x = 0; x < HD / 8; ++x) o[x][0] *= f_lo, o[x][1] *= f_lo, o[x][2] *= f_hi, o[x][3] *= f_hi;
    }
    const float z_lo = m_lo == -INFINITY ? 0.f : ac_ref<PE>(m_lo), z_hi = m_hi == -INFINITY ? 0.f : ac_ref<PE>(m_hi);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        s[n][x] = exp2f(s[n][x] - z_lo);
        s[n][2 + x] = exp2f(s[n][2 + x] - z_hi);
        l_lo += s[n][x];
        l_hi += s[n][2 + x];
      }
    // ---- O += P V ----
    landed();
    issue(2 * i + 1 + SLOTS - 1);
    const uint32_t vt = ring + ((2 * i + 1) % SLOTS) * ITEM;
    // Rows of the call's own tokens, which the tokens before them do not see, may
    // hold anything (padding): 0 times infinity would reach those.  Such rows of V
    // count as zeros, and P is NaN where a row of Q does see one (after the sum: the
    // weights do not depend on V).
    uint32_t bad = 0;
    if (w.b >= 0 && key0 + AC_KT > w.len - p.n_tok + 1 && p.n_tok > 1) {
      bad = ac_bad_rows<T, ROW>(vt, lane);
      if (bad) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int row = 8 * n + 2 * t4 + x;
            if (bad >> row & 1 && key0 + row < lim_lo) s[n][x] = NAN;
            if (bad >> row & 1 && key0 + row < lim_hi) s[n][2 + x] = NAN;
          }
      }
    }
    if constexpr (!F32) {
      // P rounded to the 16-bit type, as V is: half a step (bf16 2^-8, fp16 2^-11) of
      // each term at most, as much as the rounding of the output; the sum takes P
      // unrounded.  A second product for the rest would double those of P V.
      const uint32_t pa[4] = {pack2<T>(s[0][0], s[0][1]), pack2<T>(s[0][2], s[0][3]), pack2<T>(s[1][0], s[1][1]),
                              pack2<T>(s[1][2], s[1][3])};
      // keys 2 t4, 2 t4 + 1 and 8 more of this thread's V values
      const uint32_t k0 = bad >> (2 * t4), k1 = bad >> (8 + 2 * t4);
      const uint32_t z0 = (k0 & 1 ? 0u : 0xffffu) | (k0 & 2 ? 0u : 0xffff0000u), z1 = (k1 & 1 ? 0u : 0xffffu) | (k1 & 2 ? 0u : 0xffff0000u);
#pragma unroll
      for (int n = 0; n < HD / 16; ++n) {
        uint32_t vb[4];
        ldsm_x4_t(tile_addr<ROW>(vt, ((lane >> 3) & 1) * 8 + (lane & 7), 2 * n + (lane >> 4)), vb);
        if (bad) vb[0] &= z0, vb[1] &= z1, vb[2] &= z0, vb[3] &= z1;
        mma16<T>(o[2 * n], pa, vb[0], vb[1]);
        mma16<T>(o[2 * n + 1], pa, vb[2], vb[3]);
      }
    } else {
      // the k index t4 of step n is key 8 n + 2 t4, t4 + 4 is key 8 n + 2 t4 + 1:
      // the accumulator layout of S is the A layout of P
      uint32_t ph[2][4], pl[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        split_tf32(s[n][0], ph[n][0], pl[n][0]);
        split_tf32(s[n][2], ph[n][1], pl[n][1]);
        split_tf32(s[n][1], ph[n][2], pl[n][2]);
        split_tf32(s[n][3], ph[n][3], pl[n][3]);
      }
#pragma unroll
      for (int cg = 0; cg < HD / 32; ++cg) {
        float c[4][4];               // this tile's share, added to O in fp32 (see S)
#pragma unroll
        for (int x = 0; x < 16; ++x) c[x >> 2][x & 3] = 0.f;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          // dims 32 cg + 4 g + x are column g of n tile 4 cg + x
          float4 v0 = lds_f4(tile_addr<ROW>(vt, 8 * n + 2 * t4, 8 * cg + g));
          float4 v1 = lds_f4(tile_addr<ROW>(vt, 8 * n + 2 * t4 + 1, 8 * cg + g));
          if (bad) {
            if (bad >> (8 * n + 2 * t4) & 1) v0 = make_float4(0.f, 0.f, 0.f, 0.f);
            if (bad >> (8 * n + 2 * t4 + 1) & 1) v1 = make_float4(0.f, 0.f, 0.f, 0.f);
          }
          const float a[4] = {v0.x, v0.y, v0.z, v0.w}, b[4] = {v1.x, v1.y, v1.z, v1.w};
          uint32_t h[4][2], lo[4][2];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            split_tf32(a[x], h[x][0], lo[x][0]);
            split_tf32(b[x], h[x][1], lo[x][1]);
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) mma_tf32(c[x], ph[n], lo[x][0], lo[x][1]);
#pragma unroll
          for (int x = 0; x < 4; ++x) mma_tf32(c[x], pl[n], h[x][0], h[x][1]);
#pragma unroll
          for (int x = 0; x < 4; ++x) mma_tf32(c[x], ph[n], h[x][0], h[x][1]);
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) o[4 * cg + (x >> 2)][x & 3] += c[x >> 2][x & 3];
      }
    }
  }

  // ---- merge the key groups ----
  m_lo = ac_ref<AcType<T>::P_EXP>(m_lo);
  m_hi = ac_ref<AcType<T>::P_EXP>(m_hi);
#pragma unroll
  for (int of = 1; of <= 2; of <<= 1) {
    l_lo += __shfl_xor_sync(0xffffffffu, l_lo, of);
    l_hi += __shfl_xor_sync(0xffffffffu, l_hi, of);
  }
  if (t4 == 0) {
    s_ml[warp * 16 + g] = make_float2(m_lo, l_lo);
    s_ml[warp * 16 + g + 8] = make_float2(m_hi, l_hi);
  }
  cp_wait<0>();
  __syncthreads();                     // every group is done with Q and its ring
  float M_lo = -INFINITY, M_hi = -INFINITY;
#pragma unroll
  for (int x = 0; x < G::NG; ++x) {
    M_lo = fmaxf(M_lo, s_ml[(x * R + rt) * 16 + g].x);
    M_hi = fmaxf(M_hi, s_ml[(x * R + rt) * 16 + g + 8].x);
  }
  const float f_lo = ac_weight(make_float2(m_lo, l_lo), M_lo), f_hi = ac_weight(make_float2(m_hi, l_hi), M_hi);
  float* mo = (float*)smem + warp * 16 * HD;           // [16][HD]
  if constexpr (!F32) {
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) {
      *(float2*)(mo + g * HD + 8 * n + 2 * t4) = make_float2(o[n][0] * f_lo, o[n][1] * f_lo);
      *(float2*)(mo + (g + 8) * HD + 8 * n + 2 * t4) = make_float2(o[n][2] * f_hi, o[n][3] * f_hi);
    }
  } else {
#pragma unroll
    for (int cg = 0; cg < HD / 32; ++cg)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int d = 32 * cg + 8 * t4 + 4 * x;
        *(float4*)(mo + g * HD + d) = make_float4(o[4 * cg][x] * f_lo, o[4 * cg + 1][x] * f_lo, o[4 * cg + 2][x] * f_lo, o[4 * cg + 3][x] * f_lo);
        *(float4*)(mo + (g + 8) * HD + d) = make_float4(o[4 * cg][2 + x] * f_hi, o[4 * cg + 1][2 + x] * f_hi, o[4 * cg + 2][2 + x] * f_hi, o[4 * cg + 3][2 + x] * f_hi);
      }
  }
  __syncthreads();
  const int live = min(16 * R, w.nrows - w.row0);
#pragma unroll 4
  for (int id = tid; id < live * (HD / 4); id += G::THREADS) {
    const int r = id / (HD / 4), c = id % (HD / 4), tile = r >> 4, rr = r & 15;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < G::NG; ++x) {
      const float4 y = *(const float4*)((const float*)smem + ((x * R + tile) * 16 + rr) * HD + 4 * c);
      a.x += y.x, a.y += y.y, a.z += y.z, a.w += y.w;
    }
    const long long at = ac_entry(p, w, r);
    *(float4*)(p.part_o + at * HD + 4 * c) = a;
    if (c == 0) {
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int x = 0; x < G::NG; ++x) M = fmaxf(M, s_ml[(x * R + tile) * 16 + rr].x);
#pragma unroll
      for (int x = 0; x < G::NG; ++x) {
        const float2 y = s_ml[(x * R + tile) * 16 + rr];
        L += y.y * ac_weight(y, M);
      }
      p.part_ml[at] = make_float2(M, L);
    }
  }
}

template <typename T, int HD, int R>
__global__ void __launch_bounds__(AcGeo<T, HD, R>::THREADS, AcGeo<T, HD, R>::CTAS) ac_part_kernel(const __grid_constant__ AcParams p, AcGrid gr) {
  extern __shared__ __align__(128) uint8_t ac_smem[];
  __shared__ AcCursor s_cur;
  __shared__ AcWork s_work;
  pdl_trigger();
  if (threadIdx.x < 32) ac_first<T, HD>(p, gr, 16 * R, s_cur, s_work);
  for (;;) {
    __syncthreads();
    const AcWork w = s_work;
    if (w.j0 >= w.j1) break;
    ac_part_segment<T, HD, R>(p, w, ac_smem);
    __syncthreads();                   // the merge buffer is the next segment's ring
    if (threadIdx.x == 0) ac_next<T, HD>(p, s_cur, s_work);
  }
  // launched beside the prefix part: not complete before it, so that the
  // finishing kernel, which waits for this one, finds both
  pdl_wait();
}

// ---- fp32, few rows -------------------------------------------------------------
// A warp takes RN query rows and tiles of 32 / RN keys.  Lane l holds the dims
// 4 l .. 4 l + 3 (and 128 + those at head_dim 256) of the rows, and loads those of each key straight into registers: whole rows, coalesced, with no
// shared memory between.  The 32 partial products of a tile (keys x rows) are
// summed over the lanes by halving: at each of five steps a lane passes on half of
// its values and keeps the other half, so 31 exchanges leave lane l with the logit
// of key l / RN and row l % RN.  V's loads are in flight during S, the next K's
// during P V.  At four rows a tile of head_dim 256 takes about 400 instructions for
// 16 KB, a seventh of an SM's issue slots at the memory's rate; the tensor cores
// would spend three tf32 products of 16 rows each on it (fp32, two sequences of
// 65536 rows, four query rows: 253 us there).
constexpr int AV_WARPS = 4;

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*(unsigned long long*)&a), "l"(*(unsigned long long*)&b), "l"(*(unsigned long long*)&c));
  return *(float2*)&d;
}

template <int HD, int RN>
struct AvShared {
  float merge[AV_WARPS][RN][HD];
  float2 ml[AV_WARPS][RN];
  float q[RN][HD];
};

template <int HD, int RN>
__device__ __forceinline__ void ac_vec_segment(const AcParams& p, const AcWork w, AvShared<HD, RN>& sh) {
  constexpr int KT = 32 / RN;                      // keys of a tile
  constexpr int D2 = HD / 64;                      // float2 of a lane
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long key_stride = (long long)p.nkv * HD;
  // dims of float2 i of this lane: pairs (0, 1) and (2, 3) are one 16-byte access
  auto dim = [&](int i) { return 128 * (i >> 1) + 4 * lane + 2 * (i & 1); };
  auto load = [&](const float* src, bool ok, float2 (&x)[D2]) {
#pragma unroll
    for (int i = 0; i < D2; i += 2) {
      const float4 y = ok ? *(const float4*)(src + dim(i)) : make_float4(0.f, 0.f, 0.f, 0.f);
      x[i] = make_float2(y.x, y.y);
      x[i + 1] = make_float2(y.z, y.w);
    }
  };
  auto load_tile = [&](const uint8_t* base, int key0, float2 (&x)[KT][D2]) {
#pragma unroll
    for (int k = 0; k < KT; ++k)
      load((const float*)base + (long long)(key0 + k < w.j1 ? key0 + k : w.j0) * key_stride, key0 + k < w.j1, x[k]);
  };
  float2 kx[KT][D2], vx[KT][D2];
  int key0 = w.j0 + warp * KT;
  load_tile(w.k, key0, kx);
  load_tile(w.v, key0, vx);

  // Q in shared memory: at head_dim 128 its registers are worth more as a third
  // CTA per SM (four sequences of 30000 rows: 82 -> 74 us)
  for (int id = tid; id < RN * (HD / 4); id += AV_WARPS * 32) {
    const int r = id / (HD / 4), c = id % (HD / 4);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (w.row0 + r < w.nrows) {
      int b, t, h;
      ac_row(p, w, w.row0 + r, b, t, h);
      x = *(const float4*)((const float*)p.q + (long long)(b * p.n_tok + t) * p.q_stride + (long long)h * HD + 4 * c);
    }
    *(float4*)&sh.q[r][4 * c] = x;
  }
  __syncthreads();
  float2 o[RN][D2];
#pragma unroll
  for (int r = 0; r < RN; ++r)
#pragma unroll
    for (int i = 0; i < D2; ++i) o[r][i] = make_float2(0.f, 0.f);
  // this lane's key and row of a tile
  const int my_key = lane / RN, my_row = lane % RN;
  int lim = 0;
  float* lg = nullptr;
  if (w.row0 + my_row < w.nrows) {
    int b, t, h;
    ac_row(p, w, w.row0 + my_row, b, t, h);
    lim = w.b < 0 ? w.len : w.len - p.n_tok + 1 + t;
    if (p.scores && w.b >= 0) lg = p.logits + ((long long)(b * p.n_tok + t) * p.nh + h) * p.logit_stride;
  }
  float m = -INFINITY, l = 0.f;

  for (; key0 < w.j1; key0 += AV_WARPS * KT) {
    // ---- S = Q K^T ----
    float s[32];
#pragma unroll
    for (int r = 0; r < RN; ++r) {
      float2 q[D2];
      load(sh.q[r], true, q);
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        float2 a = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < D2; ++i) a = fma2(kx[k][i], q[i], a);
        s[k * RN + r] = a.x + a.y;
      }
    }
    load_tile(w.k, key0 + AV_WARPS * KT, kx);
#pragma unroll
    for (int st = 16; st >= 1; st >>= 1) {
      const bool up = lane & st;
#pragma unroll
      for (int i = 0; i < st; ++i) {
        const float give = up ? s[i] : s[i + st], keep = up ? s[i + st] : s[i];
        s[i] = keep + __shfl_xor_sync(0xffffffffu, give, st);
      }
    }
    // ---- running softmax of row my_row ----
    const int key = key0 + my_key;
    const float x = key < w.j1 && key < lim ? s[0] * p.scale_log2 : -INFINITY;
    if (lg && key < w.j1) lg[key] = x;
    float mx = x;
#pragma unroll
    for (int of = RN; of < 32; of <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, of));
    if (__any_sync(0xffffffffu, mx > m)) {
      const float n = fmaxf(m, mx), f = n == -INFINITY ? 1.f : exp2f(m - n);
      m = n;
      l *= f;
#pragma unroll
      for (int r = 0; r < RN; ++r) {
        const float g = __shfl_sync(0xffffffffu, f, r);
#pragma unroll
        for (int i = 0; i < D2; ++i) o[r][i].x *= g, o[r][i].y *= g;
      }
    }
    float pr = exp2f(x - (m == -INFINITY ? 0.f : m));
    l += pr;
    if (w.b >= 0 && p.n_tok > 1 && key0 + KT > w.len - p.n_tok + 1) {
      // rows of the call's own tokens: as in ac_part_kernel
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        bool is = false;
#pragma unroll
        for (int i = 0; i < D2; ++i) is |= !(fabsf(vx[k][i].x) < INFINITY) || !(fabsf(vx[k][i].y) < INFINITY);
        if (__any_sync(0xffffffffu, is)) {
#pragma unroll
          for (int i = 0; i < D2; ++i) vx[k][i] = make_float2(0.f, 0.f);
          if (my_key == k && key < lim) pr = NAN;
        }
      }
    }
    // ---- O += P V ----
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int r = 0; r < RN; ++r) {
        const float g = __shfl_sync(0xffffffffu, pr, k * RN + r);
#pragma unroll
        for (int i = 0; i < D2; ++i) o[r][i] = fma2(make_float2(g, g), vx[k][i], o[r][i]);
      }
    load_tile(w.v, key0 + AV_WARPS * KT, vx);
  }
  // ---- merge the warps ----
#pragma unroll
  for (int of = RN; of < 32; of <<= 1) l += __shfl_xor_sync(0xffffffffu, l, of);
  if (lane < RN) sh.ml[warp][lane] = make_float2(m, l);
  __syncthreads();
#pragma unroll
  for (int r = 0; r < RN; ++r) {
    float M = -INFINITY;
#pragma unroll
    for (int x = 0; x < AV_WARPS; ++x) M = fmaxf(M, sh.ml[x][r].x);
    const float f = ac_weight(sh.ml[warp][r], M);
#pragma unroll
    for (int i = 0; i < D2; ++i) *(float2*)&sh.merge[warp][r][dim(i)] = make_float2(o[r][i].x * f, o[r][i].y * f);
  }
  __syncthreads();
  const int live = min(RN, w.nrows - w.row0);
  for (int id = tid; id < live * (HD / 4); id += AV_WARPS * 32) {
    const int r = id / (HD / 4), c = id % (HD / 4);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < AV_WARPS; ++x) {
      const float4 y = *(const float4*)&sh.merge[x][r][4 * c];
      a.x += y.x, a.y += y.y, a.z += y.z, a.w += y.w;
    }
    const long long at = ac_entry(p, w, r);
    *(float4*)(p.part_o + at * HD + 4 * c) = a;
    if (c == 0) {
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int x = 0; x < AV_WARPS; ++x) M = fmaxf(M, sh.ml[x][r].x);
#pragma unroll
      for (int x = 0; x < AV_WARPS; ++x) L += sh.ml[x][r].y * ac_weight(sh.ml[x][r], M);
      p.part_ml[at] = make_float2(M, L);
    }
  }
}

template <int HD, int RN>
__global__ void __launch_bounds__(AV_WARPS * 32, HD == 256 ? 2 : 3) ac_vec_kernel(const __grid_constant__ AcParams p, AcGrid gr) {
  __shared__ AvShared<HD, RN> sh;
  __shared__ AcCursor s_cur;
  __shared__ AcWork s_work;
  pdl_trigger();
  if (threadIdx.x < 32) ac_first<float, HD>(p, gr, RN, s_cur, s_work);
  for (;;) {
    __syncthreads();
    const AcWork w = s_work;
    if (w.j0 >= w.j1) break;
    ac_vec_segment<HD, RN>(p, w, sh);
    __syncthreads();
    if (threadIdx.x == 0) ac_next<float, HD>(p, s_cur, s_work);
  }
  pdl_wait();                          // see ac_part_kernel
}

// the partials of a row: p_splits of the prefix, then those of the own part's CTAs
struct AcParts {
  long long prefix, own, step;     // first entries; between the own part's
  int n, p_splits;
  __device__ __forceinline__ long long at(int s) const { return s < p_splits ? prefix + s : own + (s - p_splits) * step; }
};
// row r of sequence b and KV head kvh (t * group + g), `row` over all
__device__ __forceinline__ AcParts ac_parts(const AcParams& p, int b, int kvh, int r, long long row) {
  AcParts x;
  x.p_splits = x.n = p.p_splits;
  x.prefix = row * p.p_splits;
  x.own = x.step = 0;
  if (p.o_groups) {
    const int nb = ac_blocks(ac_len(p, b)), tile = r / p.o_rows, units = p.nkv * p.o_tiles;
    if (nb) {
      const int share = p.head[0], pos = p.head[1 + b];
      const int c0 = pos / share, c1 = (pos + nb - 1) / share;
      x.own = p.own_base + ((long long)(c0 + b) * units + kvh * p.o_tiles + tile) * p.o_rows + (r - tile * p.o_rows);
      x.step = (long long)units * p.o_rows;
      x.n += c1 - c0 + 1;
    }
  }
  return x;
}
// (largest logit, 1 / sum) over a row's partials; called by a whole warp
__device__ __forceinline__ float2 ac_row_stats(const AcParams& p, const AcParts& parts) {
  const int lane = threadIdx.x & 31;
  float M = -INFINITY, L = 0.f;
  for (int s0 = 0; s0 < parts.n; s0 += 128) {        // 128 partials' loads in flight
    float2 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = s0 + i * 32 + lane;
      x[i] = s < parts.n ? p.part_ml[parts.at(s)] : make_float2(-INFINITY, 0.f);
    }
    const float m = warp_max(fmaxf(fmaxf(x[0].x, x[1].x), fmaxf(x[2].x, x[3].x))), n = fmaxf(M, m);
    float l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) l += x[i].y * ac_weight(x[i], n);
    L = L * ac_weight(make_float2(M, L), n) + warp_sum(l);
    M = n;
  }
  return make_float2(M, L > 0.f ? 1.f / L : (L == L ? 0.f : L));
}

// blocks [0, row_blocks): W warps per row join its splits (every W-th one each,
// then one another's sums in warp order), the loads of several in flight; blocks
// behind: `scores` of one (sequence, KV head), SLOTS own rows per thread
template <typename T, int HD, int W, int SLOTS>
__global__ void __launch_bounds__(AC_FIN_THREADS, 4) ac_finish_kernel(const __grid_constant__ AcParams p, int row_blocks, int slot_blocks) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int WARPS = AC_FIN_THREADS / 32;
  pdl_wait();
  if (blockIdx.x < row_blocks) {
    constexpr int PER = HD / 32;                     // dims of a lane
    constexpr int U = 32 / PER;                      // partials in flight
    __shared__ float part[W > 1 ? WARPS : 1][HD];
    const long long row = (long long)blockIdx.x * (WARPS / W) + warp / W;
    const long long tok = row / p.nh;
    const int h = (int)(row - tok * p.nh), sub = warp % W;
    const bool live = tok < (long long)p.batch * p.n_tok;
    if (W == 1 && !live) return;
    float a[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) a[i] = 0.f;
    float inv = 0.f;
    if (live) {
      const int b = (int)(tok / p.n_tok), t = (int)(tok - (long long)b * p.n_tok), kvh = (int)p.by_group.div(h);
      const AcParts parts = ac_parts(p, b, kvh, t * p.group + h - kvh * p.group, row);
      const int n = parts.n;
      const float2 st = ac_row_stats(p, parts);
      inv = st.y;
      const float* o = p.part_o + lane * PER;
      for (int s0 = sub; s0 < n; s0 += U * W) {
        float f[U], x[U][PER];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int s = s0 + u * W;
          f[u] = 0.f;
          if (s < n) {
            const long long at = parts.at(s);
            f[u] = ac_weight(p.part_ml[at], st.x);
#pragma unroll
            for (int i = 0; i < PER; i += 2) {
              const float2 y = *(const float2*)(o + at * HD + i);
              x[u][i] = y.x, x[u][i + 1] = y.y;
            }
          } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) x[u][i] = 0.f;
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < PER; ++i) a[i] = fmaf(f[u], x[u][i], a[i]);
      }
    }
    if constexpr (W > 1) {
#pragma unroll
      for (int i = 0; i < PER; ++i) part[warp][lane * PER + i] = a[i];
      __syncthreads();
      if (sub || !live) return;
#pragma unroll
      for (int w = 1; w < W; ++w)
#pragma unroll
        for (int i = 0; i < PER; ++i) a[i] += part[warp + w][lane * PER + i];
    }
    T* out = (T*)p.out + tok * p.out_stride + (long long)h * HD + lane * PER;
#pragma unroll
    for (int i = 0; i < PER; i += 2) {
      const float x = a[i] * inv, y = a[i + 1] * inv;
      if constexpr (AcType<T>::F32) *(float2*)(out + i) = make_float2(x, y);
      else *(uint32_t*)(out + i) = pack2<T>(x, y);
    }
    return;
  }
  constexpr int CHUNK = 64;                          // rows whose statistics are held at once
  constexpr int U = 16 / SLOTS;                      // rows whose logits are in flight
  __shared__ float2 st[CHUNK];
  __shared__ long long at[CHUNK];                    // the rows' logits
  const int x = blockIdx.x - row_blocks, bh = x / slot_blocks, b = bh / p.nkv, kvh = bh - b * p.nkv;
  const int j0 = (x - bh * slot_blocks) * (AC_FIN_THREADS * SLOTS) + threadIdx.x;
  const int len = ac_len(p, b);
  if (j0 - (int)threadIdx.x >= len) return;
  const int rows = p.n_tok * p.group;
  float sum[SLOTS];
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) sum[i] = 0.f;
  for (int r0 = 0; r0 < rows; r0 += CHUNK) {
    const int nr = min(CHUNK, rows - r0);
    // 32, 16, 8 or 4 lanes per row, so that all rows go at once
    const int tpr = nr <= WARPS ? 32 : nr <= 2 * WARPS ? 16 : nr <= 4 * WARPS ? 8 : 4;
    __syncthreads();
    {
      const int r = threadIdx.x / tpr, sub = threadIdx.x & (tpr - 1), rr = r0 + min(r, nr - 1);
      const int t = (int)p.by_group.div(rr), h = kvh * p.group + rr - t * p.group;
      const long long row = (long long)(b * p.n_tok + t) * p.nh + h;
      const AcParts parts = ac_parts(p, b, kvh, rr, row);
      float M = -INFINITY, L = 0.f;
      for (int s0 = 0; s0 < parts.n; s0 += 4 * tpr) {
        float2 y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int s = s0 + i * tpr + sub;
          y[i] = s < parts.n ? p.part_ml[parts.at(s)] : make_float2(-INFINITY, 0.f);
        }
        const float m = fmaxf(M, fmaxf(fmaxf(y[0].x, y[1].x), fmaxf(y[2].x, y[3].x)));
        float l = L * ac_weight(make_float2(M, L), m);
#pragma unroll
        for (int i = 0; i < 4; ++i) l += y[i].y * ac_weight(y[i], m);
        M = m, L = l;
      }
      for (int o = 1; o < tpr; o <<= 1) {
        const float2 y = make_float2(__shfl_xor_sync(0xffffffffu, M, o), __shfl_xor_sync(0xffffffffu, L, o));
        const float m = fmaxf(M, y.x);
        L = L * ac_weight(make_float2(M, L), m) + y.y * ac_weight(y, m);
        M = m;
      }
      if (sub == 0 && r < nr) {
        st[r] = make_float2(M, L > 0.f ? 1.f / L : (L == L ? 0.f : L));
        at[r] = row * p.logit_stride;
      }
    }
    __syncthreads();
    for (int r = 0; r < nr; r += U) {
      float lg[U][SLOTS];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
          const int j = j0 + i * AC_FIN_THREADS;
          lg[u][i] = r + u < nr && j < len ? p.logits[at[r + u] + j] : -INFINITY;
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
          if (lg[u][i] != -INFINITY) sum[i] += exp2f(lg[u][i] - st[r + u].x) * st[r + u].y;
    }
  }
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const int j = j0 + i * AC_FIN_THREADS;
    if (j < len) p.scores[(long long)bh * p.score_stride + j] += sum[i];
  }
}

// ---- host ---------------------------------------------------------------------
struct AcPlan {
  bool p_tc;                      // prefix part on tcgen05 (ap_rows() rows per CTA)
  int p_r, o_r;                   // rows per CTA of the two parts: 16, 32, 64 (ac_part_kernel), 4, 8 (ac_vec_kernel)
  int p_tiles;                    // row tiles of the prefix part
  long long rows;                 // query rows over all heads
  size_t off_ml, off_head, off_logits, bytes;
};

// Rows per CTA for a part with `rows` query rows per KV head and `len` keys.  fp32
// with few rows goes to ac_vec_kernel in tiles of 4 or 8, where the tensor cores'
// three products cost more than the lanes' sums: head_dim 256 up to 8 rows (two
// sequences of 15000 to 30000: 78 us against 107), or 16 over few keys, which end
// sooner there (prefix of 500: 12.6 us against 14.3; 30000: 97 against 85); 128 up to
// 4 (four such sequences: 66 against 78; 8 rows: 107 against 79); not 64 (4 rows of
// 30000: 69 against 58).
int ac_row_class(int type, int hd, long long rows, int len) {
  if (type == INFERNO_F32 && rows <= (hd == 256 ? (len <= 4096 ? 16 : 8) : hd == 128 ? 4 : 0)) return rows <= 4 ? 4 : 8;
  return rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}

// Splits of the prefix when `units` (KV heads x row tiles) share the GPU, of which
// at_once CTAs run at a time: as many as fill one to four rounds of CTAs, whichever
// ends first when a CTA takes the time of its keys and of `start` more.  (Against
// splits of 256 keys in any number of rounds, fp32: 32 query rows of head_dim 256 x 4
// heads on 16000 keys, 252 CTAs of 256 -> 144 of 448, 90 -> 76 us; 64 rows on 4096,
// 64 -> 56; head_dim 128, 16 rows x 8 heads on 20000, 58 -> 46.)  A split has min_len
// keys at least.
void ac_split(long long units, long long at_once, long long len, long long min_len, long long start, AcParams* p) {
  double best = 0;
  p->p_splits = 0;
  for (int rounds = 1; rounds <= 4; ++rounds) {
    const long long want = std::max(1ll, std::min(256ll, rounds * at_once / units));
    const long long keys = std::max(min_len, ((len + want - 1) / want + 63) / 64 * 64), splits = (len + keys - 1) / keys;
    const double time = (double)((splits * units + at_once - 1) / at_once) * (double)(keys + start);
    if (p->p_splits && time >= best) continue;
    best = time;
    p->p_split_len = (int)keys;
    p->p_splits = (int)splits;
  }
}

template <typename T, int HD>
int ac_ctas_per_sm(int r) {
  if (r <= 8) return HD == 256 ? 2 : 3;                    // ac_vec_kernel
  return r == 16 ? AcGeo<T, HD, 1>::CTAS : r == 32 ? AcGeo<T, HD, 2>::CTAS : AcGeo<T, HD, 4>::CTAS;
}
int ac_ctas_per_sm(int type, int hd, int r) {
  if (type == INFERNO_F32)
    return hd == 64 ? ac_ctas_per_sm<float, 64>(r) : hd == 128 ? ac_ctas_per_sm<float, 128>(r) : ac_ctas_per_sm<float, 256>(r);
  return hd == 64 ? ac_ctas_per_sm<__half, 64>(r) : hd == 128 ? ac_ctas_per_sm<__half, 128>(r) : ac_ctas_per_sm<__half, 256>(r);
}

// The prefix part of a 16-bit type on tcgen05 or on mma.sync.  tcgen05 takes 128 rows
// at a time, but starts later (TMEM, barriers) and at head_dim 64 waits for its
// exponentials.  mma.sync with up to 16 rows, its one row tile, streams as fast; above
// that by the number of products (rows in tiles of 16 x keys x KV heads x head_dim).
// Whole calls, bf16, tcgen05 / mma.sync, us:
//   head_dim 64, 4 heads: 32 rows x 16000 15.3 / 13.4 (x 60000, 8 heads 41 / 46), 48 x
//   4000 10.9 / 10.5, 64 x 4000 11.4 / 12.2, 48 x 16000 15.4 / 18.1
//   128: 16 x 16000 17.1 / 15.4 (x 60000, 8 heads 49 / 49), 32 x 1000 10.4 / 9.2, 48 x
//   1000 10.4 / 10.6, 32 x 4000 11.1 / 13.1
//   256: 16 x 16000 24.5 / 23.6, 48 x 300 12.0 / 15.8, 32 x 1000 13.1 / 13.3, 32 x 4000
//   15.3 / 21.1
bool ac_prefix_tc(const InfernoAttention* a, long long rows) {
  if (a->type == INFERNO_F32 || rows <= 16) return false;
  const double products = (double)((rows + 15) / 16 * 16) * a->prefix_len * a->n_kv_heads * a->head_dim;
  return products >= (a->head_dim == 64 ? (rows > 32 ? 60e6 : 300e6) : a->head_dim == 128 ? 20e6 : 12e6);
}

int ac_check(const InfernoAttention* a) {
  if (!a) return set_error(INFERNO_EINVAL, "attention_cached: null parameters");
  if (a->struct_size && a->struct_size != (int)sizeof(InfernoAttention))
    return set_error(INFERNO_EINVAL, "attention_cached: struct_size %d, expected %d", a->struct_size,
                     (int)sizeof(InfernoAttention));
  if (!longctx_type_size(a->type))
    return set_error(INFERNO_EINVAL, "attention_cached: type %d is not F32, F16 or BF16", a->type);
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256)
    return set_error(INFERNO_EINVAL, "attention_cached: head_dim %d is not 64, 128 or 256", a->head_dim);
  if (a->batch < 0 || a->n_tokens < 1 || a->n_heads < 1 || a->n_kv_heads < 1 || a->n_heads % a->n_kv_heads)
    return set_error(INFERNO_EINVAL, "attention_cached: bad sizes (batch %d, %d tokens, %d / %d heads)", a->batch,
                     a->n_tokens, a->n_heads, a->n_kv_heads);
  if (a->prefix_len < 0 || a->max_len < 0)
    return set_error(INFERNO_EINVAL, "attention_cached: prefix_len %d, max_len %d", a->prefix_len, a->max_len);
  if (a->prefix_len > (1 << 30) || a->max_len > (1 << 30) || a->n_heads > 65536 ||
      (double)a->batch * a->n_tokens * a->n_heads > (double)(1 << 24))
    return set_error(INFERNO_EINVAL, "attention_cached: more than 2^24 query rows or 2^30 keys");
  if ((double)a->batch * (a->max_len / AC_BLOCK + 1) > (double)(1 << 30))
    return set_error(INFERNO_EINVAL, "attention_cached: more than 2^30 blocks of %d keys", AC_BLOCK);
  if (!std::isfinite(a->scale)) return set_error(INFERNO_EINVAL, "attention_cached: scale is not finite");
  return 0;
}

AcPlan ac_plan(const InfernoAttention* a, AcParams* p) {
  AcPlan pl{};
  p->batch = a->batch;
  p->n_tok = a->n_tokens;
  p->nh = a->n_heads;
  p->nkv = a->n_kv_heads;
  p->group = a->n_heads / a->n_kv_heads;
  p->prefix_len = a->prefix_len;
  p->max_len = a->max_len;
  p->by_seq = FastDiv((uint32_t)(a->n_tokens * p->group));
  p->by_group = FastDiv((uint32_t)p->group);
  const long long own = (long long)a->n_tokens * p->group, pre = own * a->batch;
  pl.rows = pre * a->n_kv_heads;
  pl.o_r = ac_row_class(a->type, a->head_dim, own, a->max_len);
  pl.p_r = ac_row_class(a->type, a->head_dim, pre, a->prefix_len);
  // both parts in one launch where the own part is small beside the prefix and
  // can take the prefix part's kernel: a launch costs more than idle rows then
  if (a->prefix_len && a->max_len && pl.p_r > pl.o_r && (pl.p_r <= 8 || pl.o_r >= 16) && !ac_prefix_tc(a, pre) &&
      (long long)a->max_len * a->batch <= a->prefix_len)
    pl.o_r = pl.p_r;
  p->o_rows = pl.o_r;
  p->o_tiles = (int)((own + pl.o_r - 1) / pl.o_r);
  pl.p_tiles = (int)((pre + pl.p_r - 1) / pl.p_r);
  p->p_splits = 0;
  pl.p_tc = ac_prefix_tc(a, pre);
  if (!a->prefix_len) {
  } else if (pl.p_tc) {
    // starting and joining a CTA takes about as long as eight tiles (13 row tiles x 8
    // heads on 8000 keys: 101 us in one round of 208 CTAs, 90 in two of 520)
    pl.p_tiles = (int)((pre + ap_rows() - 1) / ap_rows());
    ac_split((long long)pl.p_tiles * a->n_kv_heads, (long long)AC_SMS * ap_ctas_per_sm(a->head_dim), a->prefix_len, 128,
             512, p);
  } else {
    // one tile of 16 for each of four key groups at least
    ac_split((long long)pl.p_tiles * a->n_kv_heads, (long long)AC_SMS * ac_ctas_per_sm(a->type, a->head_dim, pl.p_r),
             a->prefix_len, 64, 96, p);
  }
  // own part: as many groups of CTAs as fit the GPU at once (two rounds where a
  // group is large, whose remainder would idle), a block of keys each at least.
  // Long shares are cut finer, a round more per 32 blocks up to four: the SMs do
  // not stream alike, and what the early ones save outweighs more starts and merges
  // (16 bf16 sequences of up to 16384 rows, 110 blocks: 157 us in one round, 152 in
  // three; two f32 ones of 65536, 28 blocks: 116 in one and 132 in three).
  const long long units = (long long)a->n_kv_heads * p->o_tiles;
  const long long blocks = (long long)a->batch * ((a->max_len + AC_BLOCK - 1) / AC_BLOCK);
  const long long at_once = (long long)AC_SMS * ac_ctas_per_sm(a->type, a->head_dim, pl.o_r);
  long long groups = units <= at_once / 8 ? at_once / units : (2 * at_once + units - 1) / units;
  groups *= std::max(1ll, std::min(4ll, blocks / (32 * groups)));
  p->o_groups = (int)std::min(blocks, groups);
  p->by_groups = FastDiv((uint32_t)std::max(1, p->o_groups));
  p->own_base = pl.rows * p->p_splits;
  const long long entries = p->own_base + (p->o_groups ? (p->o_groups + a->batch) * units * pl.o_r : 0);
  p->logit_stride = a->scores ? ((long long)a->max_len + 15) / 16 * 16 : 0;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  pl.off_ml = up((size_t)entries * a->head_dim * 4);
  pl.off_head = pl.off_ml + up((size_t)entries * 8);
  pl.off_logits = pl.off_head + up((size_t)(1 + a->batch) * 4);
  pl.bytes = pl.off_logits + up((size_t)pl.rows * p->logit_stride * 4) + 256;
  return pl;
}

// beside: may start while the kernel before it in the call still runs (it waits
// for that one itself)
template <typename... Args, typename... Given>
cudaError_t ac_launch(void (*kernel)(Args...), long long blocks, int threads, size_t smem, cudaStream_t st, bool beside,
                      Given... args) {
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = beside ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T, int HD, int R>
cudaError_t ac_launch_part(const AcParams& p, AcGrid gr, long long blocks, bool beside, cudaStream_t st) {
  using G = AcGeo<T, HD, R>;
  static DeviceOnce once;
  cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(ac_part_kernel<T, HD, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM);
  });
  if (e != cudaSuccess) return e;
  return ac_launch(ac_part_kernel<T, HD, R>, blocks, G::THREADS, G::SMEM, st, beside, p, gr);
}
// one kernel over the prefix part, the own part or both, r rows per CTA
template <typename T, int HD>
cudaError_t ac_part(const AcParams& p, const AcPlan& pl, int r, bool prefix, bool own, bool beside, cudaStream_t st) {
  const long long pb = prefix ? (long long)pl.p_tiles * p.nkv * p.p_splits : 0;
  const long long blocks = pb + (own ? (long long)p.o_groups * p.nkv * p.o_tiles : 0);
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  const AcGrid gr{(int)pb, pl.p_tiles};
  if constexpr (AcType<T>::F32 && HD >= 128) {
    if (r == 4) return ac_launch(ac_vec_kernel<HD, 4>, blocks, AV_WARPS * 32, 0, st, beside, p, gr);
  }
  if constexpr (AcType<T>::F32 && HD == 256) {
    if (r == 8) return ac_launch(ac_vec_kernel<HD, 8>, blocks, AV_WARPS * 32, 0, st, beside, p, gr);
  }
  return r == 16   ? ac_launch_part<T, HD, 1>(p, gr, blocks, beside, st)
         : r == 32 ? ac_launch_part<T, HD, 2>(p, gr, blocks, beside, st)
                   : ac_launch_part<T, HD, 4>(p, gr, blocks, beside, st);
}
template <typename T, int HD>
cudaError_t ac_run(const AcParams& p, const AcPlan& pl, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  bool any = pl.p_tc && p.p_splits;    // a kernel of this call is in flight
  const bool prefix = p.p_splits && !pl.p_tc, own = p.o_groups > 0;
  if (prefix && own && pl.p_r == pl.o_r) {
    e = ac_part<T, HD>(p, pl, pl.p_r, true, true, false, st);
    any = true;
  } else {
    if (prefix) {
      e = ac_part<T, HD>(p, pl, pl.p_r, true, false, false, st);
      any = true;
    }
    if (e == cudaSuccess && own) {
      e = ac_part<T, HD>(p, pl, pl.o_r, false, true, any, st);
      any = true;
    }
  }
  if (e != cudaSuccess) return e;
  // warps per row by its partials, one warp having 4 to 16 in flight; the own part's
  // are about as many as groups per sequence
  const long long parts = p.p_splits + (p.o_groups ? 1 + p.o_groups / p.batch : 0);
  const int warps = parts <= 8 ? 1 : parts <= 24 ? 4 : 8;
  const int per_block = AC_FIN_THREADS / 32 / warps;
  const long long row_blocks = (pl.rows + per_block - 1) / per_block;
  // four cache rows per thread, or one where that leaves fewer than two CTAs per SM
  const long long heads = (long long)p.batch * p.nkv;
  const int slots = p.scores && heads * ((p.max_len + 4 * AC_FIN_THREADS - 1) / (4 * AC_FIN_THREADS)) >= 2 * AC_SMS ? 4 : 1;
  const long long slot_blocks = p.scores ? (p.max_len + slots * AC_FIN_THREADS - 1) / (slots * AC_FIN_THREADS) : 0;
  const long long blocks = row_blocks + slot_blocks * heads;
  auto* kernel = slots == 4 ? (warps == 1 ? ac_finish_kernel<T, HD, 1, 4> : warps == 4 ? ac_finish_kernel<T, HD, 4, 4> : ac_finish_kernel<T, HD, 8, 4>)
                            : (warps == 1 ? ac_finish_kernel<T, HD, 1, 1> : warps == 4 ? ac_finish_kernel<T, HD, 4, 1> : ac_finish_kernel<T, HD, 8, 1>);
  return ac_launch(kernel, blocks, AC_FIN_THREADS, 0, st, any, p, (int)row_blocks, (int)std::max(1ll, slot_blocks));
}
template <typename T>
cudaError_t ac_run_hd(int hd, const AcParams& p, const AcPlan& pl, cudaStream_t st) {
  return hd == 64 ? ac_run<T, 64>(p, pl, st) : hd == 128 ? ac_run<T, 128>(p, pl, st) : ac_run<T, 256>(p, pl, st);
}

}  // namespace
}  // namespace inf

using namespace inf;

extern "C" int64_t inferno_attention_cached_workspace(const InfernoAttention* a) {
  const int rc = ac_check(a);
  if (rc) return rc;
  if (a->batch == 0) return 256;              // nothing to plan for
  AcParams p{};
  return (int64_t)ac_plan(a, &p).bytes;
}

namespace {

int ac_call(const InfernoAttention* a, void* workspace, int64_t workspace_bytes, void* stream, bool give_up) {
  int rc = ac_check(a);
  if (rc) return rc;
  if (a->batch == 0) return 0;
  const long long es = longctx_type_size(a->type), row = (long long)a->n_kv_heads * a->head_dim;
  const long long qrow = (long long)a->n_heads * a->head_dim;
  if (!a->q || !a->out) return set_error(INFERNO_EINVAL, "attention_cached: q or out missing");
  if (a->prefix_len && (!a->prefix_k || !a->prefix_v))
    return set_error(INFERNO_EINVAL, "attention_cached: prefix_k or prefix_v missing");
  if (a->max_len && (!a->k_cache || !a->v_cache || !a->lens))
    return set_error(INFERNO_EINVAL, "attention_cached: k_cache, v_cache or lens missing");
  if ((long long)a->batch * a->n_tokens > 1 && (a->q_stride < qrow || a->out_stride < qrow))
    return set_error(INFERNO_EINVAL, "attention_cached: q_stride %lld or out_stride %lld is less than a token row of %lld",
                     (long long)a->q_stride, (long long)a->out_stride, qrow);
  if (a->max_len && a->batch > 1 && a->seq_stride < row * a->max_len)
    return set_error(INFERNO_EINVAL, "attention_cached: seq_stride %lld is less than a slice of %d rows",
                     (long long)a->seq_stride, a->max_len);
  if (a->scores && (long long)a->batch * a->n_kv_heads > 1 && a->score_stride < a->max_len)
    return set_error(INFERNO_EINVAL, "attention_cached: score_stride %lld is less than max_len %d",
                     (long long)a->score_stride, a->max_len);
  uintptr_t al = (uintptr_t)a->q | (uintptr_t)a->out | (uintptr_t)(a->q_stride * es) | (uintptr_t)(a->out_stride * es);
  if (a->prefix_len) al |= (uintptr_t)a->prefix_k | (uintptr_t)a->prefix_v;
  if (a->max_len) al |= (uintptr_t)a->k_cache | (uintptr_t)a->v_cache | (uintptr_t)(a->seq_stride * es);
  if (al % 16) return set_error(INFERNO_EINVAL, "attention_cached: a pointer or stride is not a multiple of 16 bytes");
  if (((uintptr_t)a->lens | (uintptr_t)a->scores) % 4)
    return set_error(INFERNO_EINVAL, "attention_cached: lens or scores is not a multiple of 4 bytes");
  AcParams p{};
  const AcPlan pl = ac_plan(a, &p);
  if (give_up && !(pl.p_tc && p.p_splits))
    return set_error(INFERNO_EINVAL, "attention_cached: no bounded waits in a call of these sizes");
  if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < (int64_t)pl.bytes)
    return set_error(INFERNO_EINVAL, "attention_cached: workspace of %lld bytes, %lld needed (256-byte aligned)",
                     (long long)workspace_bytes, (long long)pl.bytes);
  if ((rc = longctx_check_device({a->q, a->out, workspace}, "attention_cached"))) return rc;
  if (a->prefix_len && (rc = longctx_check_device({a->prefix_k, a->prefix_v}, "attention_cached"))) return rc;
  if (a->max_len && (rc = longctx_check_device({a->k_cache, a->v_cache, a->lens, a->scores}, "attention_cached"))) return rc;
  p.q = a->q;
  p.pk = a->prefix_k;
  p.pv = a->prefix_v;
  p.kc = a->k_cache;
  p.vc = a->v_cache;
  p.lens = a->lens;
  p.out = a->out;
  p.scores = a->max_len ? a->scores : nullptr;
  p.q_stride = a->q_stride;
  p.out_stride = a->out_stride;
  p.seq_stride = a->batch > 1 ? a->seq_stride : 0;
  p.score_stride = a->score_stride;
  p.scale_log2 = (a->scale == 0.0f ? 1.0f / sqrtf((float)a->head_dim) : a->scale) * AC_LOG2E;
  p.part_o = (float*)workspace;
  p.part_ml = (float2*)((char*)workspace + pl.off_ml);
  p.head = (int*)((char*)workspace + pl.off_head);
  p.logits = (float*)((char*)workspace + pl.off_logits);
  cudaStream_t st = (cudaStream_t)stream;
  if (pl.p_tc && p.p_splits && (rc = launch_attn_prefix_tc(a->type, a->head_dim, p, pl.p_tiles, give_up, st))) return rc;
  const cudaError_t e = a->type == INFERNO_F32   ? ac_run_hd<float>(a->head_dim, p, pl, st)
                        : a->type == INFERNO_F16 ? ac_run_hd<__half>(a->head_dim, p, pl, st)
                                                 : ac_run_hd<__nv_bfloat16>(a->head_dim, p, pl, st);
  return e == cudaSuccess ? 0 : set_error(INFERNO_ECUDA, "attention_cached launch: %s", cudaGetErrorString(e));
}

}  // namespace

extern "C" int inferno_attention_cached(const InfernoAttention* a, void* workspace, int64_t workspace_bytes,
                                        void* stream) {
  return ac_call(a, workspace, workspace_bytes, stream, false);
}

extern "C" int inferno_debug_attention_timeout(const InfernoAttention* a, void* workspace, int64_t workspace_bytes,
                                               void* stream) {
  return ac_call(a, workspace, workspace_bytes, stream, true);
}
