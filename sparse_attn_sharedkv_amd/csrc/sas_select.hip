// Choosing the rows that sparse attention reads (no reference counterpart: the reference takes
// cmp_sparse_indices as an input, api.py:137, and its tests draw them at random,
// golden.py:411-473).
//
// For a query row t at causal position p = act_kv - act_q + s of its sequence, every compressed
// row j < thr = floor((p + 1) / cmp_ratio) has the score
//   s(t, j) = scale_j * sum_h w[t, h] * max(0, q[t, h] . k[j])          (scale_j = 1 without fp8)
// and the ids of the topk largest are written in ascending order, -1 behind them; among equal
// scores the lowest ids win. Rows on a page outside the pool are never chosen.
//
// Two kernels. The first forms fp32 scores with MFMA and writes them to the workspace; the
// second, a workgroup for each row, finds the topk-th largest and writes the ids.
//
// Which rows are chosen does not depend on how the scores were summed. An fp32 score is off by at
// most E = c W K, c = (D + H / 16 + 8) 2^-23, W = sum_h |w_h| |q_h|, K = max_j |k_j| (below), so a row
// whose fp32 score is more than 2 E above the topk-th largest fp32 score is in, one more than 2 E
// below it is out, and the few in between are scored again in 64 bits. Ids are therefore those
// of 64-bit scores for any split of the work, any batch and any tile.
//
// The bound. Products of two 16-bit numbers are exact in fp32. A dot product's D terms are added
// in some order and with some grouping inside the matrix instruction; each addition loses at most
// 2^-23 of the sum of the magnitudes (a rounding 2^-24, a truncated alignment twice that), so it
// is off by at most D 2^-23 sum |q_i k_i| <= D 2^-23 |q| |k|. max(0, x) moves no two values
// further apart. A weighted term passes through at most H / 8 + 1 fused steps of one of eight
// chains, three sums that join them and an fp8 row's scale, 2^-24 of the magnitudes each:
// (H / 16 + 2.5) 2^-23. The rest of c is slack for terms of second order and for the norms' own
// rounding. 2^-50 is added to each norm for products below fp32's normal range. A bound that is
// not finite (infinities, NaN, norms beyond fp32) has the whole row scored in 64 bits.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/sas_mi355x.h"
#include "sas_items.h"

namespace sas {

void set_error(const std::string& msg);

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr float SEL_NONE = -__builtin_inff();  // score of a row that cannot be chosen
constexpr float SEL_MAX = 3.402823466e38f;     // scores are kept inside [-SEL_MAX, SEL_MAX]
constexpr float SEL_TINY = 8.8817841970012523e-16f;  // 2^-50

template <typename T>
struct Elem;
template <>
struct Elem<__bf16> {
  typedef bf16x8 v8;
  static __device__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ float dot2(uint32_t a, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a),
                                           __builtin_bit_cast(bf16x2, a), c, false);
  }
  // two e4m3 codes (the low or the high half of w), scaled by 1
  static __device__ uint32_t widen(uint32_t w, bool high) {
    return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
  }
  static __device__ float lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
  static __device__ float hi(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
};
template <>
struct Elem<_Float16> {
  typedef f16x8 v8;
  static __device__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ float dot2(uint32_t a, float c) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, a), __builtin_bit_cast(f16x2, a), c,
                                  false);
  }
  static __device__ uint32_t widen(uint32_t w, bool high) {
    return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
  }
  static __device__ float lo(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[0]; }
  static __device__ float hi(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[1]; }
};

// Eight e4m3 codes as eight elements of T (exact: e4m3 fits in both 16-bit types).
template <typename T>
__device__ inline u32x4 widen_e4m3(u32x2 c) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    r[2 * i] = Elem<T>::widen(c[i], false);
    r[2 * i + 1] = Elem<T>::widen(c[i], true);
  }
  return r;
}

// The bound on an fp32 score's error: 0 where every score is exactly 0 (no weights, or keys without
// a bit set: a cache nobody has written), infinite where it says nothing. 2^-110 is above what sums and products below fp32's normal range lose.
__device__ inline float score_error(const SasSelectArgs& a, float w_norm, float k_norm2) {
  if (w_norm == 0.0f || k_norm2 == 0.0f) return 0.0f;
  const float err = ((float)a.dim + (float)a.heads / 16.0f + 8.0f) * 1.1920929e-7f * w_norm *
                    (sqrtf(k_norm2) + SEL_TINY);
  return err <= SEL_MAX ? fmaxf(err, 7.7037197775489434e-34f) : __builtin_inff();
}

// Sequences of fewer query rows than this have their keys read for each row.
constexpr int SEL_FEW_ROWS = 4;

// How a score kernel shares a row's keys out.
struct SelSplit {
  int chunks;  // workgroups that share a row's keys
  int slices;  // waves that share a piece's keys
  int norms;   // key norms that a piece leaves (one of each wave that has looked at keys)
};

// What the kernels know of a launch besides its arguments.
struct SelPlan {
  int t_begin, t_end;   // query rows of this pass
  int width;            // scores kept for a row (row stride of the workspace)
  int few_rows;         // sequences of fewer rows than this go to score_stream_kernel
  SelSplit few, many;   // of score_stream_kernel, of score_tile_kernel
  int norm_stride;      // key norms of a sequence
  FastDiv page_div, ratio_div;
  float* w_norm;        // [rows of the pass] W of each row
  float* k_norm;        // [batch][norm_stride] largest |k|^2 of the keys seen
  float* score;         // [rows of the pass][width]
};

struct RowPos {
  int b;     // sequence, -1: a row of no sequence
  int thr;   // keys the row may choose from
  int last;  // first query row behind the sequence's (or behind the run of rows of no sequence)
  int rows;  // query rows of the sequence
};

__device__ inline RowPos locate(const SasSelectArgs& a, const SelPlan& p, int t) {
  RowPos r;
  int s, act_q;
  if (a.rows_per_seq > 0) {
    const int b = t / a.rows_per_seq;
    s = t - b * a.rows_per_seq;
    act_q = a.cu_seqlens_q ? a.cu_seqlens_q[b + 1] - a.cu_seqlens_q[b] : a.rows_per_seq;
    if (act_q > a.rows_per_seq) act_q = a.rows_per_seq;
    if (s >= act_q) return {-1, 0, (b + 1) * a.rows_per_seq, 0};
    r.b = b;
    r.last = b * a.rows_per_seq + act_q;
  } else {
    // the last sequence that starts at or before row t (empty ones before it start there too);
    // where every sequence has one row that is sequence t
    int lo = -1, hi = a.batch;  // cu[lo] <= t < cu[hi]
    if (t < a.batch && a.cu_seqlens_q[t] <= t && t < a.cu_seqlens_q[t + 1]) {
      lo = t;
      hi = t + 1;
    }
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu_seqlens_q[mid] <= t) {
        lo = mid;
      } else {
        hi = mid;
      }
    }
    if (lo < 0) return {-1, 0, a.batch > 0 ? a.cu_seqlens_q[0] : a.tokens, 0};
    const int first = a.cu_seqlens_q[lo], end = a.cu_seqlens_q[lo + 1];
    if (t >= end) return {-1, 0, lo + 1 < a.batch ? a.cu_seqlens_q[lo + 1] : a.tokens, 0};
    r.b = lo;
    s = t - first;
    act_q = end - first;
    r.last = end;
  }
  const ItemGeom g = item_geom_div(act_q, a.seqused_kv[r.b], s, -1, 2, p.ratio_div, 0);
  r.thr = min(g.thr, a.max_keys);
  r.rows = act_q;
  return r;
}

__device__ inline int thr_at(const SasSelectArgs& a, const SelPlan& p, int t) {
  return locate(a, p, t).thr;
}

// Keys of one of a row's pieces: equal shares of the keys it has, in whole steps of 64 keys a
// slice, so no workgroup of a short sequence in a wide table goes without work before the
// last pieces do.
__device__ inline int piece_keys(const SelSplit& sp, int thr) {
  const int unit = 64 * sp.slices;
  return ((thr + sp.chunks - 1) / sp.chunks + unit - 1) / unit * unit;
}

// ---------------------------------------------------------------------------
// Scores
// ---------------------------------------------------------------------------
//
// Q is the A operand (rows are heads), keys the B operand (columns are keys), so a lane ends with
// 16 heads of one key and the weighted sum over heads is a chain of fmas in registers and one
// exchange between the wave's halves. A query row's Q (2 KB a head block and K step) and weights
// stay in registers for all of a wave's keys.
//
// The K dimension is taken in an order that gives a lane whole runs of a key row: step 2 p + u,
// half hf of the wave holds dims [32 p + 16 hf + 8 u, +8) of both operands.

// max(0, x), in one instruction (a float's bits order like a signed integer's at zero; fmaxf
// takes two, the first to quiet what NaN there may be; positive NaN stays NaN here)
__device__ inline float above_zero(float x) {
  return __builtin_bit_cast(float, max(__builtin_bit_cast(int, x), 0));
}

__device__ inline int frag_dim(int p, int u, int hf) { return 32 * p + 16 * hf + 8 * u; }

// The weights are in registers too (W_LDS = 0), or in a wave's own piece of LDS.
template <typename T, int D, int MT, bool W_LDS>
struct QueryFrags {
  u32x4 q[MT][D / 16];
  f32x16 w[W_LDS ? 1 : MT];
  float* w_lds;  // [32 MT]

  __device__ void load(const SasSelectArgs& a, int t, int lane) {
    const int m = lane & 31, hf = lane >> 5;
    const T* base = (const T*)a.q + (int64_t)t * a.heads * D;
    const float* wb = a.weights + (int64_t)t * a.heads;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      // (heads there are not: the last one's, with weight 0)
      const int h = min(32 * mt + m, a.heads - 1);
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        q[mt][k] = *(const u32x4*)(base + (int64_t)h * D + frag_dim(k >> 1, k & 1, hf));
      if (W_LDS) {
        const float v = wb[h];
        if (hf == 0) w_lds[32 * mt + m] = 32 * mt + m < a.heads ? v : 0.0f;
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int hh = 32 * mt + 8 * (i >> 2) + 4 * hf + (i & 3);
          const float v = wb[min(hh, a.heads - 1)];
          w[W_LDS ? 0 : mt][i] = hh < a.heads ? v : 0.0f;
        }
      }
    }
  }

  // sum_h |w_h| (|q_h| + 2^-50), the same in every lane
  __device__ float bound(const SasSelectArgs& a, int t, int lane) const {
    float s = 0.0f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float n2 = 0.0f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = Elem<T>::lo(q[mt][k][e]), y = Elem<T>::hi(q[mt][k][e]);
          n2 = fmaf(x, x, fmaf(y, y, n2));
        }
      n2 += __shfl_xor(n2, 32, 64);
      const int h = 32 * mt + (lane & 31);
      if (h < a.heads) {
        const float w = fabsf(a.weights[(int64_t)t * a.heads + h]);
        const float v = w * (sqrtf(n2) + SEL_TINY);
        s += w != 0.0f && v < 7.52e-37f ? 7.52e-37f : v;  // (2^-120: no weight but 0 vanishes)
      }
    }
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) s += __shfl_xor(s, off, 64);
    return s;
  }

  // the score of key lane & 31 without its scale
  __device__ float score(const u32x4 k[D / 16], int hf) const {
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      f32x16 acc = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) acc = Elem<T>::mfma(q[mt][kk], k[kk], acc);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float wv[4];
        if (W_LDS) {
          const float4 v = *(const float4*)(w_lds + 32 * mt + 8 * g + 4 * hf);
          wv[0] = v.x, wv[1] = v.y, wv[2] = v.z, wv[3] = v.w;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) wv[i] = w[W_LDS ? 0 : mt][4 * g + i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = fmaf(above_zero(acc[4 * g + i]), wv[i], s[i]);
      }
    }
    const float r = (s[0] + s[1]) + (s[2] + s[3]);
    return r + __shfl_xor(r, 32, 64);
  }
};

// |k|^2, or the smallest normal number where a key that is not 0 has no square in fp32.
__device__ inline float norm_kept(float n2, bool zero) { return n2 == 0.0f && !zero ? 1.17549435e-38f : n2; }

template <typename T, int D>
__device__ inline float key_norm2(const u32x4 k[D / 16], float scale) {
  float n[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
    for (int e = 0; e < 4; ++e) n[e] = Elem<T>::dot2(k[kk][e], n[e]);
  float s = (n[0] + n[1]) + (n[2] + n[3]);
  s += __shfl_xor(s, 32, 64);
  s *= scale * scale;
  if (__any(s == 0.0f)) {
    uint32_t bits = 0;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) bits |= k[kk][0] | k[kk][1] | k[kk][2] | k[kk][3];
    bits |= __shfl_xor(bits, 32, 64);
    s = norm_kept(s, (bits & 0x7fff7fffu) == 0 || scale == 0.0f);
  }
  return s;
}

__device__ inline float kept_score(float s) {
  // NaN ranks lowest; the bound is not finite then, nor where a score leaves fp32's range
  return s == s ? fminf(fmaxf(s, -SEL_MAX), SEL_MAX) : -SEL_MAX;
}

// Larger of two non-negative numbers, where NaN is above infinity.
__device__ inline float max_nonneg(float a, float b) {
  return __builtin_bit_cast(float, max(__builtin_bit_cast(uint32_t, a) & 0x7fffffffu,
                                       __builtin_bit_cast(uint32_t, b) & 0x7fffffffu));
}

// Byte offset in LDS of 16-byte chunk c of row r, C chunks to a row: the rows' chunks are rotated
// against each other, so that 16 lanes reading one chunk of 16 rows touch every bank once.
template <int C>
__device__ inline int chunk_at(int r, int c) {
  return r * (16 * C) + ((c ^ (r / (16 / C) & (C - 1))) << 4);
}

// Decode: few query rows a sequence. A workgroup's four waves take a quarter each of a piece of one
// query row's keys, and share nothing: no barrier. Whole key rows come from memory into registers
// (a lane's own parts of its key would be 32 short runs a load), through a wave's own LDS into the
// operand's layout, and the next tiles' are on their way under the current one's products.
// Bound by the keys' bytes. Measured with 64 heads of 128 dims: 64 rows over 32768 bf16 keys
// 118 us, 4.5 TB/s (the loads alone, nothing formed of them, 102 us); 128 rows over 32768 to
// 131072 fp8 keys 357 us, 3.9 TB/s (alone 300 us). Rows of one sequence read its keys once each:
// a second row's come out of L2 (64 x 2 rows: 171 us).
// Tiles in flight: fp8 2, 3 or 1 took 357, 373 and 458 us (3 spill at 64 heads), bf16 1 or 2 took
// 110 and 122 us.
constexpr int STREAM_WAVES = 4;

template <bool FP8>
constexpr int STREAM_DEPTH = FP8 ? 2 : 1;  // tiles of 32 keys that a wave has on their way

template <typename T, bool FP8, int D, int MT>
__global__ __launch_bounds__(64 * STREAM_WAVES, MT <= 2 ? 2 : 1) void score_stream_kernel(SasSelectArgs a, SelPlan p) {
  __shared__ __attribute__((aligned(256))) unsigned char stage[STREAM_WAVES][32 * (FP8 ? D : 2 * D)];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 31, hf = lane >> 5;
  const int piece = (int)(blockIdx.x % (unsigned)p.few.chunks);
  int t = (int)(blockIdx.x / (unsigned)p.few.chunks);
  if (p.few_rows == SEL_FEW_ROWS) {
    // a mixed step: the workgroups are of the rows that short sequences may have
    const int b = t / (SEL_FEW_ROWS - 1), s = t - b * (SEL_FEW_ROWS - 1);
    const int first = a.cu_seqlens_q[b], rows = a.cu_seqlens_q[b + 1] - first;
    if (s >= rows || rows >= SEL_FEW_ROWS) return;
    t = s + (a.rows_per_seq > 0 ? b * a.rows_per_seq : first);
    if (t < p.t_begin || t >= p.t_end) return;
  } else {
    t += p.t_begin;
  }
  const RowPos r = locate(a, p, t);
  const int keys = piece_keys(p.few, r.thr), lo = piece * keys;
  if (r.b < 0 || r.rows >= p.few_rows || r.thr <= a.topk || lo >= r.thr) return;
  const int hi = min(lo + keys, r.thr), slice = wave, step = 32 * STREAM_WAVES;

  QueryFrags<T, D, MT, false> qf;
  qf.load(a, t, lane);
  if (piece == 0 && slice == 0) {
    const float w = qf.bound(a, t, lane);
    if (lane == 0) p.w_norm[t - p.t_begin] = w;
  }
  const bool norms = t == min(r.last, p.t_end) - 1;
  float kn = 0.0f;
  const int32_t* table = a.block_table + (int64_t)r.b * a.table_len;
  float* out = p.score + (int64_t)(t - p.t_begin) * p.width;

  // DEPTH tiles on their way from memory, and the pages of the DEPTH behind them
  constexpr int ROW = FP8 ? D : 2 * D, LOADS = ROW / 32, DEPTH = STREAM_DEPTH<FP8>;
  constexpr int C = ROW / 16, R = 64 / C;  // 16-byte chunks of a row, rows of a load
  const uint32_t page_units = (uint32_t)((int64_t)a.block_size * (FP8 ? D + 4 : 2 * D) / 16);
  const unsigned char* lane_keys = (const unsigned char*)a.keys + 16 * (lane % C);
  unsigned char* own = stage[wave];
  u32x4 raw[DEPTH][LOADS];
  float scale[DEPTH];
  bool ok[DEPTH];
  int page[DEPTH];
  auto page_of = [&](int j) { return j < hi ? table[p.page_div.div(j)] : -1; };
  auto load = [&](int u, int j) {
    ok[u] = page[u] >= 0 && page[u] < a.block_num;
    const uint32_t at = ok[u] ? j - p.page_div.div(j) * a.block_size : 0;
    const uint32_t pg = (ok[u] ? (uint32_t)page[u] : 0) * page_units;
    // where the lane's key starts, in 16 bytes (the pool has fewer than 2^32 of them)
    const int unit = (int)(pg + at * C);
#pragma unroll
    for (int q = 0; q < LOADS; ++q) {
      const uint32_t from = (uint32_t)__shfl(unit, R * q + lane / C, 64);
      raw[u][q] = *(const u32x4*)(lane_keys + (uint64_t)from * 16);
    }
    if (FP8) {
      scale[u] = *(const float*)((const unsigned char*)a.keys + (uint64_t)(pg + (uint32_t)a.block_size * C) * 16 +
                                 4 * at);
    }
  };
  // whole rows into LDS as they came, a lane's parts of its key out of it (a wave's own piece of
  // LDS: its accesses keep their order)
  auto turn = [&](int u, u32x4 part[LOADS]) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int q = 0; q < LOADS; ++q)
      *(u32x4*)(own + chunk_at<C>(R * q + lane / C, lane % C)) = raw[u][q];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      // fp8: 16 codes, the steps 2 i and 2 i + 1
      const int c = FP8 ? 2 * i + hf : frag_dim(i >> 1, i & 1, hf) / 8;
      part[i] = *(const u32x4*)(own + chunk_at<C>(n, c));
    }
  };

  const int first = lo + 32 * slice;
#pragma unroll
  for (int u = 0; u < DEPTH; ++u) page[u] = page_of(first + u * step + n);
#pragma unroll
  for (int u = 0; u < DEPTH; ++u) {
    load(u, first + u * step + n);
    page[u] = page_of(first + (DEPTH + u) * step + n);
  }
  u32x4 part[LOADS];
  if (FP8 && first < hi) turn(0, part);
  for (int base = first; base < hi; base += DEPTH * step) {
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) {
      const int j = base + u * step + n;
      if (base + u * step >= hi) break;
      const float sc = FP8 ? scale[u] : 1.0f;
      const bool is = ok[u];
      if (!FP8) turn(u, part);
      load(u, j + DEPTH * step);
      page[u] = page_of(j + 2 * DEPTH * step);
      u32x4 k[D / 16];
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        if (FP8) {
          k[2 * i] = widen_e4m3<T>(u32x2{part[i][0], part[i][1]});
          k[2 * i + 1] = widen_e4m3<T>(u32x2{part[i][2], part[i][3]});
        } else {
          k[i] = part[i];
        }
      }
      if (FP8) turn((u + 1) % DEPTH, part);  // the next tile's, under this one's products
      if (norms) {
        const float n2 = key_norm2<T, D>(k, sc);
        if (is) kn = max_nonneg(kn, n2);
      }
      float s = qf.score(k, hf);
      if (FP8) s *= sc;
      if (hf == 0 && j < hi) out[j] = is ? kept_score(s) : SEL_NONE;
    }
  }
  if (norms) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) kn = max_nonneg(kn, __shfl_xor(kn, off, 64));
    if (lane == 0) p.k_norm[(int64_t)r.b * p.norm_stride + piece * p.few.norms + slice] = kn;
  }
}

// Prefill: many query rows a sequence. A workgroup's eight waves own one query row each and
// share the keys, 64 at a time through LDS (two stages there, two more on their way in registers;
// fp8 codes are widened on the way in). Bound by the matrix cores and, as much, by the weighted
// sums: a 32-key tile of 64 heads is 16 matrix instructions (512 cycles) and some 120 vector ones
// (480), which two waves a SIMD overlap only in part (matrix cores busy 40 %, vector units 40 %).
// 8192 causal rows over 2048 keys, 64 heads of 128 dims: 149 us, 870 TFLOP/s. Four waves and
// 32 keys a stage, twice the workgroups a CU: 172 us; instruction groups forced to alternate: 167.
// A tile of eight rows that spans sequences takes them one after the other.
constexpr int TILE_WAVES = 8;
constexpr int TILE_KEYS = 64;

template <typename T, bool FP8, int D, int MT>
__global__ __launch_bounds__(64 * TILE_WAVES) void score_tile_kernel(SasSelectArgs a, SelPlan p) {
  __shared__ __attribute__((aligned(256))) unsigned char stage[2][TILE_KEYS * D * 2];
  __shared__ float key_scale[2][TILE_KEYS];
  __shared__ int key_ok[2][TILE_KEYS];
  __shared__ __attribute__((aligned(16))) float weight[TILE_WAVES][32 * MT];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 31, hf = lane >> 5;
  const int piece = (int)(blockIdx.x % (unsigned)p.many.chunks);
  const int tiles = (p.t_end - p.t_begin + TILE_WAVES - 1) / TILE_WAVES;
  // the last rows of a causal prefill have the most keys: they start first
  const int t0 = p.t_begin + (tiles - 1 - (int)(blockIdx.x / (unsigned)p.many.chunks)) * TILE_WAVES;
  const int t1 = min(t0 + TILE_WAVES, p.t_end), t = t0 + wave;
  // the thread's part of a stage: bytes [32 part, +32) of native row `row`, or 16 codes
  constexpr int PARTS = 64 * TILE_WAVES / TILE_KEYS;   // 8 threads a row
  constexpr int LOADS = FP8 ? 1 : D * 2 / (16 * PARTS);  // 16-byte loads of a thread
  const int row = threadIdx.x / PARTS, part = threadIdx.x % PARTS;
  const bool loads_codes = !FP8 || part < D / 16;

  QueryFrags<T, D, MT, true> qf;
  qf.w_lds = weight[wave];
  for (int ts = t0; ts < t1;) {
    const RowPos seg = locate(a, p, ts);
    const int te = max(min(seg.last, t1), ts + 1);
    const int thr_end = seg.b < 0 || seg.rows < p.few_rows ? 0 : thr_at(a, p, te - 1);
    const int keys = piece_keys(p.many, thr_end), lo = piece * keys, hi = min(lo + keys, thr_end);
    if (thr_end <= a.topk || lo >= thr_end) {
      ts = te;
      continue;
    }
    const bool mine = t >= ts && t < te;
    const int my_thr = mine ? thr_at(a, p, t) : 0;
    const bool active = mine && my_thr > a.topk && lo < my_thr;
    const bool norms = te == min(seg.last, p.t_end);  // the tile that sees all of the sequence's keys
    if (active) {
      qf.load(a, t, lane);
      if (piece == 0) {
        const float w = qf.bound(a, t, lane);
        if (lane == 0) p.w_norm[t - p.t_begin] = w;
      }
    }
    const int32_t* table = a.block_table + (int64_t)seg.b * a.table_len;
    float* out = p.score + (int64_t)(t - p.t_begin) * p.width;
    float kn = 0.0f;

    // two stages on their way: in registers until the one before them has been read
    u32x4 held[2][LOADS];
    float held_scale[2] = {1.0f, 1.0f};
    int held_ok[2], page[2];
    auto page_of = [&](int j) { return j < hi ? table[p.page_div.div(j)] : -1; };
    auto fetch = [&](int u, int j) {
      held_ok[u] = page[u] >= 0 && page[u] < a.block_num;
      const int at = held_ok[u] ? j - p.page_div.div(j) * a.block_size : 0;
      const int64_t pg = held_ok[u] ? page[u] : 0;
      if (!FP8) {
        const unsigned char* src = (const unsigned char*)a.keys + (pg * a.block_size + at) * (2 * D);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) held[u][i] = *(const u32x4*)(src + 16 * (part * LOADS + i));
      } else {
        const unsigned char* src = (const unsigned char*)a.keys + pg * a.block_size * (D + 4);
        if (loads_codes) held[u][0] = *(const u32x4*)(src + at * D + 16 * part);
        held_scale[u] = *(const float*)(src + (int64_t)a.block_size * D + 4 * at);
      }
    };
    auto put = [&](int buf) {
      if (norms) {
        u32x4 k[2] = {};
        if (!FP8) {
#pragma unroll
          for (int i = 0; i < LOADS; ++i) k[i] = held[buf][i];
        } else if (loads_codes) {
          k[0] = widen_e4m3<T>(u32x2{held[buf][0][0], held[buf][0][1]});
          k[1] = widen_e4m3<T>(u32x2{held[buf][0][2], held[buf][0][3]});
        }
        float n2 = 0.0f;
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            n2 = Elem<T>::dot2(k[i][e], n2);
            bits |= k[i][e];
          }
#pragma unroll
        for (int off = 1; off < PARTS; off <<= 1) {
          n2 += __shfl_xor(n2, off, 64);
          bits |= __shfl_xor(bits, off, 64);
        }
        if (FP8) n2 *= held_scale[buf] * held_scale[buf];
        n2 = norm_kept(n2, (bits & 0x7fff7fffu) == 0 || (FP8 && held_scale[buf] == 0.0f));
        if (held_ok[buf]) kn = max_nonneg(kn, n2);
      }
      if (!FP8) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
          *(u32x4*)(stage[buf] + chunk_at<D / 8>(row, part * LOADS + i)) = held[buf][i];
      } else if (loads_codes) {
        *(u32x4*)(stage[buf] + chunk_at<D / 8>(row, 2 * part)) =
            widen_e4m3<T>(u32x2{held[buf][0][0], held[buf][0][1]});
        *(u32x4*)(stage[buf] + chunk_at<D / 8>(row, 2 * part + 1)) =
            widen_e4m3<T>(u32x2{held[buf][0][2], held[buf][0][3]});
      }
      if (part == 0) {
        key_ok[buf][row] = held_ok[buf];
        key_scale[buf][row] = held_scale[buf];
      }
    };

#pragma unroll
    for (int u = 0; u < 2; ++u) page[u] = page_of(lo + TILE_KEYS * u + row);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      fetch(u, lo + TILE_KEYS * u + row);
      page[u] = page_of(lo + TILE_KEYS * (2 + u) + row);
    }
    put(0);
    __syncthreads();
    for (int base2 = lo; base2 < hi; base2 += 2 * TILE_KEYS) {
#pragma unroll
      for (int buf = 0; buf < 2; ++buf) {
        const int base = base2 + TILE_KEYS * buf;
        if (base >= hi) break;
        fetch(buf, base + 2 * TILE_KEYS + row);
        page[buf] = page_of(base + 4 * TILE_KEYS + row);
        if (active) {
          // both halves of the stage without a branch between them, so that one's weighted sums
          // can run under the other's products; then each half of the wave keeps 32 scores
          float s = 0.0f;
#pragma unroll(MT *D <= 256 ? TILE_KEYS / 32 : 1)
          for (int kt = 0; kt < TILE_KEYS / 32; ++kt) {
            u32x4 k[D / 16];
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              k[kk] = *(const u32x4*)(stage[buf] + chunk_at<D / 8>(32 * kt + n, frag_dim(kk >> 1, kk & 1, hf) / 8));
            const float part = qf.score(k, hf);
            s = hf == kt ? part : s;
          }
          if (FP8) s *= key_scale[buf][lane];
          const int j = base + lane;
          if (j < my_thr && j < hi) out[j] = key_ok[buf][lane] ? kept_score(s) : SEL_NONE;
        }
        if (base + TILE_KEYS < hi) put(buf ^ 1);
        __syncthreads();
      }
    }
    if (norms) {
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) kn = max_nonneg(kn, __shfl_xor(kn, off, 64));
      if (lane == 0) p.k_norm[(int64_t)seg.b * p.norm_stride + piece * p.many.norms + wave] = kn;
    }
    ts = te;
  }
}

// ---------------------------------------------------------------------------
// Selection
// ---------------------------------------------------------------------------
//
// A workgroup for each query row. The row's scores (or, of a row too long for the registers, the
// ones above a threshold that a sample puts a little below the topk-th) are in registers:
//   1. the topk-th largest, by one histogram over their range and a ranking inside its bin;
//   2. those above the bound are taken, those inside it scored in 64 bits and ranked;
//   3. every id taken is a bit of a map in LDS, from which the ids come out in order.
// Bound by the latency of these steps, not by bytes, so steps are few and long rows get many
// waves, while the many short rows of a prefill get one wave each, which needs no barriers. Of the
// 36 us that a row of some 80000 scores takes (128 of them at once), its length, bound and sample
// are 6, the list 12, the topk-th and what is near it 6, 64-bit scores and ranks of the 49 rows
// inside the bound 11, the ids 1.5.
// What does not fit (a bound that is not finite, more equal scores than the lists hold) goes
// through select_from_memory: the same steps over the scores in memory, as often as it takes.

template <int THREADS>
struct SelSize {
  static constexpr int WAVES = THREADS / 64;
  static constexpr int BINS = THREADS == 64 ? 512 : THREADS == 256 ? 1024 : 2048;
  static constexpr int LIST = THREADS == 64 ? 128 : THREADS == 256 ? 256 : 1024;
  static constexpr int PARTS = THREADS == 64 ? 1 : SAS_SELECT_MAX_HEADS / 16;
};

// The workgroup's sums take one barrier each: every use has a row of SelShared::sums of its own.
enum SelSlot { SLOT_THERE, SLOT_SAMPLE, SLOT_COUNT, SLOT_ABOVE, SLOT_IDS, SLOT_NUM };

template <int THREADS>
struct SelShared {
  typedef SelSize<THREADS> S;
  uint32_t bins[S::BINS];
  float list_x[S::LIST];
  int list_j[S::LIST];
  uint64_t list_key[S::LIST];
  int sums[SLOT_NUM][S::WAVES];
  int wave_a[S::WAVES], wave_b[S::WAVES];
  float wave_lo[S::WAVES], wave_hi[S::WAVES];
  int close_j[S::LIST];
  int count, found, below, in_bin, sure, close;
  float value;
};

__device__ inline uint64_t order_of(double s) {
  // larger score, larger number; NaN as the lowest, -0 as 0
  if (!(s == s)) s = -__builtin_inf();
  s += 0.0;
  const uint64_t u = __builtin_bit_cast(uint64_t, s);
  return u >> 63 ? ~u : u | (1ull << 63);
}

// Scores of 16 keys over 16 heads in 64 bits, by one wave: lane l is key l & 15 (`j`, any id of the
// sequence) and holds a quarter of the dims of it and of head h0 + (l & 15), so that both operands
// come in whole 16-byte loads; the dims are summed in the order the matrix instruction takes
// them. Returns the heads' weighted sum for the lane's key without its scale, the same in its four
// lanes. Element r of the product is head 4 r + l / 16.
template <typename T, bool FP8>
__device__ inline double score64_part(const SasSelectArgs& a, const SelPlan& p, int t,
                                      const int32_t* table, int j, int h0, int lane) {
  const int d = a.dim, quarter = d / 4, c = lane & 15, kq = lane >> 4;
  const int pg = p.page_div.div(j);
  int64_t page = table[pg], at = j - pg * a.block_size;
  if (page < 0 || page >= a.block_num) page = at = 0;  // (a key nobody asks for)
  const int h = h0 + c;
  const T* q = (const T*)a.q + ((int64_t)t * a.heads + min(h, a.heads - 1)) * d + kq * quarter;
  u32x4 qv[4], kv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (8 * i < quarter) qv[i] = *(const u32x4*)(q + 8 * i);
  }
  if (!FP8) {
    const T* k = (const T*)a.keys + (page * a.block_size + at) * d + kq * quarter;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (8 * i < quarter) kv[i] = *(const u32x4*)(k + 8 * i);
    }
  } else {
    const unsigned char* k = (const unsigned char*)a.keys + page * a.block_size * (d + 4) + at * d +
                             kq * quarter;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (8 * i < quarter) kv[i] = widen_e4m3<T>(*(const u32x2*)(k + 8 * i));
    }
  }
  double w[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int hh = h0 + 4 * r + kq;
    w[r] = hh < a.heads ? (double)a.weights[(int64_t)t * a.heads + hh] : 0.0;
  }
  f64x4 acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (8 * i >= quarter) break;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)Elem<T>::lo(qv[i][e]),
                                                 (double)Elem<T>::lo(kv[i][e]), acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)Elem<T>::hi(qv[i][e]),
                                                 (double)Elem<T>::hi(kv[i][e]), acc, 0, 0, 0);
    }
  }
  double s = 0.0;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const double x = acc[r] < 0.0 ? 0.0 : acc[r];  // (keeps NaN)
    if (h0 + 4 * r + kq < a.heads) s += x * w[r];
  }
  s += __shfl_xor(s, 16, 64);
  return s + __shfl_xor(s, 32, 64);
}

template <bool FP8>
__device__ inline double key_scale64(const SasSelectArgs& a, const SelPlan& p, const int32_t* table,
                                     int j) {
  if (!FP8) return 1.0;
  const int pg = p.page_div.div(j), at = j - pg * a.block_size;
  const int64_t page = table[pg];
  if (page < 0 || page >= a.block_num) return 0.0;
  return (double)*(const float*)((const unsigned char*)a.keys + page * a.block_size * (a.dim + 4) +
                                 (int64_t)a.block_size * a.dim + 4 * at);
}

// Order of the scores of 16 keys (lane l: key `j`, l & 15), by one wave.
template <typename T, bool FP8>
__device__ inline uint64_t order64(const SasSelectArgs& a, const SelPlan& p, int t,
                                   const int32_t* table, int j, int lane) {
  double s = 0.0;
  for (int h0 = 0; h0 < a.heads; h0 += 16) s += score64_part<T, FP8>(a, p, t, table, j, h0, lane);
  return order_of(s * key_scale64<FP8>(a, p, table, j));
}

// Reductions over a wave on the vector ALU (data-parallel shifts; lane 63 ends with the result).
template <typename F>
__device__ inline int wave_scan(int v, int identity, F op) {
  v = op(v, __builtin_amdgcn_update_dpp(identity, v, 0x111, 0xf, 0xf, false));  // row_shr:1
  v = op(v, __builtin_amdgcn_update_dpp(identity, v, 0x112, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(identity, v, 0x114, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(identity, v, 0x118, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(identity, v, 0x142, 0xa, 0xf, false));  // row_bcast:15
  return op(v, __builtin_amdgcn_update_dpp(identity, v, 0x143, 0xc, 0xf, false));  // row_bcast:31
}
__device__ inline int as_int(float f) { return __builtin_bit_cast(int, f); }
__device__ inline float as_float(int i) { return __builtin_bit_cast(float, i); }
__device__ inline int wave_incl(int v) {
  return wave_scan(v, 0, [](int a, int b) { return a + b; });
}
__device__ inline int wave_sum(int v) { return __builtin_amdgcn_readlane(wave_incl(v), 63); }
__device__ inline float wave_min(float v) {
  const int r = wave_scan(as_int(v), as_int(SEL_MAX), [](int a, int b) {
    return as_int(fminf(as_float(a), as_float(b)));
  });
  return as_float(__builtin_amdgcn_readlane(r, 63));
}
__device__ inline float wave_max(float v) { return -wave_min(-v); }


template <int THREADS>
__device__ inline int block_sum(int v, SelSlot slot, SelShared<THREADS>& sh) {
  v = wave_sum(v);
  if (THREADS == 64) return v;
  if ((threadIdx.x & 63) == 0) sh.sums[slot][threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) v += sh.sums[slot][w];
  return v;
}

// Sum of the threads' values before this one's; `all` is the sum of every thread's.
template <int THREADS>
__device__ inline int block_before(int v, SelSlot slot, SelShared<THREADS>& sh, int& all) {
  const int incl = wave_incl(v);
  if (THREADS == 64) {
    all = __builtin_amdgcn_readlane(incl, 63);
    return incl - v;
  }
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 63) sh.sums[slot][wave] = incl;
  __syncthreads();
  int before = incl - v;
  all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    before += w < wave ? sh.sums[slot][w] : 0;
    all += sh.sums[slot][w];
  }
  return before;
}

// The range of the workgroup's values, the same in every thread.
template <int THREADS>
__device__ inline void block_range(float& lo, float& hi, SelShared<THREADS>& sh) {
  lo = wave_min(lo);
  hi = wave_max(hi);
  if (THREADS == 64) return;
  __syncthreads();  // (its two rows have several uses)
  if ((threadIdx.x & 63) == 0) {
    sh.wave_lo[threadIdx.x >> 6] = lo;
    sh.wave_hi[threadIdx.x >> 6] = hi;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    lo = fminf(lo, sh.wave_lo[w]);
    hi = fmaxf(hi, sh.wave_hi[w]);
  }
}

// Finds the bin that holds the need-th value from the top: sh.found, the values above it
// sh.below, and its own sh.in_bin. Ends with a barrier.
template <int THREADS>
__device__ inline void find_bin(int need, SelSlot slot, SelShared<THREADS>& sh) {
  constexpr int BINS = SelSize<THREADS>::BINS, PER = BINS / THREADS;
  int c[PER], sum = 0, all;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    c[i] = (int)sh.bins[BINS - 1 - ((int)threadIdx.x * PER + i)];
    sum += c[i];
  }
  int before = block_before<THREADS>(sum, slot, sh, all);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (before < need && need <= before + c[i]) {
      sh.found = BINS - 1 - ((int)threadIdx.x * PER + i);
      sh.below = before;
      sh.in_bin = c[i];
    }
    before += c[i];
  }
  __syncthreads();
}

// A monotone map of [lo, hi] onto the bins.
template <int THREADS>
struct BinMap {
  float base, inv;
  __device__ static BinMap of(float lo, float hi) {
    return {0.5f * lo, (float)(SelSize<THREADS>::BINS - 1) / (0.5f * hi - 0.5f * lo)};
  }
  __device__ bool usable() const { return inv < SEL_MAX; }
  // lo <= x <= hi: 0.5 x - base is in [0, 0.5 hi - base], its product below BINS
  __device__ int bin(float x) const { return (int)(fmaf(0.5f, x, -base) * inv); }
  __device__ float edge(int bin) const { return 2.0f * ((float)bin / inv + base); }  // about
};

// The choice from scores in memory, for what the registers and lists do not hold.
template <typename T, bool FP8, int THREADS>
__device__ inline void select_from_memory(const SasSelectArgs& a, const SelPlan& p, int t, int n,
                                          float err, float* x_of, const int32_t* table,
                                          SelShared<THREADS>& sh) {
  constexpr int WAVES = THREADS / 64, BINS = SelSize<THREADS>::BINS, LIST = SelSize<THREADS>::LIST;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int k = a.topk;
  int32_t* ids = a.out + (int64_t)t * k;

  // Ids of the rows that `taken` says, in order: each wave owns a run of the row, counts what it
  // takes, and writes behind the waves before it. Of the rows that `tied` says the first
  // `ties` in order are taken too.
  const int run = ((n + WAVES - 1) / WAVES + 63) & ~63;
  const int j0 = wave * run, j1 = min(j0 + run, n);
  auto emit = [&](auto taken, auto tied, int ties) {
    int mine = 0, eq = 0;
    for (int j = j0; j < j1; j += 64) {
      const int jj = j + lane;
      const bool in = jj < j1;
      mine += __popcll(__ballot(in && taken(jj)));
      eq += __popcll(__ballot(in && tied(jj)));
    }
    __syncthreads();
    if (lane == 0) {
      sh.wave_a[wave] = mine;
      sh.wave_b[wave] = eq;
    }
    __syncthreads();
    int at = 0, all = 0, eq_before = 0, eqs_all = 0;
    for (int w = 0; w < WAVES; ++w) {
      if (w == wave) {
        at = all;
        eq_before = eqs_all;
      }
      all += sh.wave_a[w] + max(min(sh.wave_b[w], ties - eqs_all), 0);
      eqs_all += sh.wave_b[w];
    }
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    for (int j = j0; j < j1; j += 64) {
      const int jj = j + lane;
      const bool in = jj < j1;
      const bool is_eq = in && tied(jj);
      const uint64_t eqs = __ballot(is_eq);
      const bool take = (in && taken(jj)) || (is_eq && eq_before + __popcll(eqs & below) < ties);
      const uint64_t takes = __ballot(take);
      const int pos = at + __popcll(takes & below);
      if (take && pos < k) ids[pos] = jj;
      at += __popcll(takes);
      eq_before += __popcll(eqs);
    }
    for (int i = all + tid; i < k; i += THREADS) ids[i] = -1;
  };

  float lo = SEL_MAX, hi = -SEL_MAX;
  int there = 0, edge = 0;
  for (int j = tid; j < n; j += THREADS) {
    const float x = x_of[j];
    if (x != SEL_NONE) {
      lo = fminf(lo, x);
      hi = fmaxf(hi, x);
      ++there;
      edge |= fabsf(x) >= SEL_MAX;
    }
  }
  block_range<THREADS>(lo, hi, sh);
  __syncthreads();
  there = block_sum<THREADS>(there, SLOT_THERE, sh);
  edge = block_sum<THREADS>(edge, SLOT_ABOVE, sh);
  if (edge) err = __builtin_inff();
  if (there <= k) {
    emit([&](int j) { return x_of[j] != SEL_NONE; }, [](int) { return false; }, 0);
    return;
  }

  // [lo, hi] around the k-th largest fp32 score: linear bins over the range, then over the bin
  // that holds it, until it is known or the range cannot be cut any more
  int need = k;
  while (lo < hi) {
    const BinMap<THREADS> map = BinMap<THREADS>::of(lo, hi);
    if (!map.usable()) break;
    auto bin_of = [&](float x) { return map.bin(x); };
    __syncthreads();
    for (int i = tid; i < BINS; i += THREADS) sh.bins[i] = 0;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    for (int j = tid; j < n; j += THREADS) {
      const float x = x_of[j];
      if (x >= lo && x <= hi) atomicAdd(&sh.bins[bin_of(x)], 1u);
    }
    __syncthreads();
    find_bin<THREADS>(need, SLOT_COUNT, sh);
    const int bin = sh.found, in_bin = sh.in_bin;
    need -= sh.below;
    if (in_bin <= LIST) {
      for (int j = tid; j < n; j += THREADS) {
        const float x = x_of[j];
        if (x >= lo && x <= hi && bin_of(x) == bin) sh.list_x[atomicAdd(&sh.count, 1)] = x;
      }
      __syncthreads();
      for (int i = tid; i < in_bin; i += THREADS) {
        const float x = sh.list_x[i];
        int above = 0, same = 0;
        for (int m = 0; m < in_bin; ++m) {
          above += sh.list_x[m] > x;
          same += sh.list_x[m] == x;
        }
        if (above < need && need <= above + same) sh.value = x;
      }
      __syncthreads();
      lo = hi = sh.value;
      break;
    }
    float l2 = SEL_MAX, h2 = -SEL_MAX;
    for (int j = tid; j < n; j += THREADS) {
      const float x = x_of[j];
      if (x >= lo && x <= hi && bin_of(x) == bin) {
        l2 = fminf(l2, x);
        h2 = fmaxf(h2, x);
      }
    }
    block_range<THREADS>(l2, h2, sh);
    if (l2 == lo && h2 == hi) break;
    lo = l2;
    hi = h2;
  }

  // rows within the bound of the k-th largest
  const bool exact = err == 0.0f && lo == hi;
  const float b_lo = exact ? lo : lo - 2.0f * err, b_hi = exact ? hi : hi + 2.0f * err;
  __syncthreads();
  if (tid == 0) sh.count = 0;
  __syncthreads();
  int sure = 0;
  for (int j = tid; j < n; j += THREADS) {
    const float x = x_of[j];
    sure += x > b_hi;
    if (x >= b_lo && x <= b_hi && x != SEL_NONE) {
      const int i = atomicAdd(&sh.count, 1);
      if (i < LIST) sh.list_j[i] = j;
    }
  }
  sure = block_sum<THREADS>(sure, SLOT_SAMPLE, sh);
  __syncthreads();
  const int close = sh.count, rest = k - sure;  // `rest` of the `close` rows are taken
  if (exact) {
    emit([&](int j) { return x_of[j] > hi; }, [&](int j) { return x_of[j] == hi; }, rest);
    return;
  }
  if (close == rest) {
    emit([&](int j) { return x_of[j] >= b_lo && x_of[j] != SEL_NONE; }, [](int) { return false; }, 0);
    return;
  }
  const float taken_x = __builtin_inff();
  if (close <= LIST) {
    for (int i = 16 * wave; i < close; i += 16 * WAVES) {
      const int e = min(i + (lane & 15), close - 1);
      const uint64_t key = order64<T, FP8>(a, p, t, table, sh.list_j[e], lane);
      if (lane < 16 && i + lane < close) sh.list_key[i + lane] = key;
    }
    __syncthreads();
    for (int i = tid; i < close; i += THREADS) {
      const uint64_t key = sh.list_key[i];
      const int j = sh.list_j[i];
      int rank = 0;
      for (int m = 0; m < close; ++m) {
        const uint64_t o = sh.list_key[m];
        rank += o > key || (o == key && sh.list_j[m] < j);
      }
      x_of[j] = rank < rest ? taken_x : SEL_NONE;
    }
    __syncthreads();
    const float above = fminf(b_hi, SEL_MAX);
    emit([&](int j) { return x_of[j] > above; }, [](int) { return false; }, 0);
    return;
  }
  // more of them than the list holds (equal keys, or a bound that is not finite): the rest-th
  // largest 64-bit score digit by digit. A row whose digits so far are not those of that score is
  // marked taken or not and is not scored again, so the most rows are scored two or three times.
  constexpr int DIGIT = THREADS == 64 ? 9 : THREADS == 256 ? 10 : 11;  // 2^DIGIT bins
  const float tie_x = SEL_MAX;
  uint64_t prefix = 0;
  int want = rest;
  for (int j = tid; j < n; j += THREADS) {
    const float x = x_of[j];
    if (x > b_hi) {
      x_of[j] = taken_x;
    } else if (!(x >= b_lo) || x == SEL_NONE) {
      x_of[j] = SEL_NONE;
    } else {
      x_of[j] = tie_x;  // (as far as is known)
    }
  }
  for (int seen = 0; seen < 64; seen += DIGIT) {
    const int left = 64 - seen, digit_bits = left < DIGIT ? left : DIGIT, shift = left - digit_bits;
    for (int i = tid; i < BINS; i += THREADS) sh.bins[i] = 0;
    __syncthreads();
    for (int j0 = 16 * wave; j0 < n; j0 += 16 * WAVES) {
      const int j = min(j0 + (lane & 15), n - 1);
      const bool tied = x_of[j] == tie_x;
      if (!__any(tied)) continue;
      const uint64_t key = order64<T, FP8>(a, p, t, table, j, lane);
      if (lane < 16 && tied && j0 + lane < n) {
        const uint64_t head = seen == 0 ? 0 : key >> left;
        if (head == prefix) {
          atomicAdd(&sh.bins[(key >> shift) & ((1u << digit_bits) - 1)], 1u);
        } else {
          x_of[j] = head > prefix ? taken_x : SEL_NONE;
        }
      }
    }
    __syncthreads();
    find_bin<THREADS>(want, SLOT_COUNT, sh);
    want -= sh.below;
    prefix = (prefix << digit_bits) | (uint64_t)sh.found;
    __syncthreads();
  }
  for (int j0 = 16 * wave; j0 < n; j0 += 16 * WAVES) {
    const int j = min(j0 + (lane & 15), n - 1);
    const bool tied = x_of[j] == tie_x;
    if (!__any(tied)) continue;
    const uint64_t key = order64<T, FP8>(a, p, t, table, j, lane);
    if (lane < 16 && tied && j0 + lane < n && key != prefix) x_of[j] = key > prefix ? taken_x : SEL_NONE;
  }
  __syncthreads();
  emit([&](int j) { return x_of[j] > SEL_MAX; }, [&](int j) { return x_of[j] == tie_x; }, want);
}

// Rows longer than this have no place in the map of select_kernel's ids.
constexpr int SEL_SAMPLED_KEYS = 1 << 18;

// Eight bits to every fourth bit.
__device__ inline uint32_t every_fourth(uint32_t b) {
  b = (b | (b << 12)) & 0x000f000fu;
  b = (b | (b << 6)) & 0x03030303u;
  return (b | (b << 3)) & 0x11111111u;
}

// Where the rank of `count` listed values (larger first, equal ones by id) is `want`, says so.
template <int THREADS, typename K, typename F>
__device__ inline void rank_list(int count, const K* key, const int* id, F at) {
  constexpr int SHARE = THREADS == 64 ? 1 : 16;  // lanes that rank one value
  for (int i = threadIdx.x / SHARE; i < count; i += THREADS / SHARE) {
    const K x = key[i];
    const int j = id[i];
    int rank = 0;
#pragma unroll 4
    for (int e = threadIdx.x % SHARE; e < count; e += SHARE) {
      const K y = key[e];
      rank += y > x || (y == x && id[e] < j);
    }
#pragma unroll
    for (int off = 1; off < SHARE; off <<= 1) rank += __shfl_xor(rank, off, 64);
    if (threadIdx.x % SHARE == 0) at(i, rank);
  }
}

// SAMPLED: rows of any length, of which at most CAP scores get into registers; else rows of at
// most CAP. Value i of a thread is id (i / 4) 4 THREADS + 4 tid + i % 4 (whole 16 bytes, side by
// side in a wave), or what the list of a long row has.
template <typename T, bool FP8, int THREADS, int VPT, bool SAMPLED>
__global__ __launch_bounds__(THREADS, THREADS == 64 ? 5 : 4) void select_kernel(SasSelectArgs a, SelPlan p) {
  constexpr int WAVES = THREADS / 64, BINS = SelSize<THREADS>::BINS, LIST = SelSize<THREADS>::LIST;
  constexpr int CAP = THREADS * VPT, MAP = SAMPLED ? SEL_SAMPLED_KEYS / 32 : CAP / 32;
  struct Listed {
    float x[SAMPLED ? CAP : 1];
    int id[SAMPLED ? CAP : 1];
  };
  __shared__ SelShared<THREADS> sh;
  // taken ids. A listed row: id j is bit j. Else in the order the waves vote: a run of 256 ids has
  // four numbers of 64 bits, bit l of number c is the run's id 4 l + c
  __shared__ __attribute__((aligned(16))) uint32_t map[MAP];
  __shared__ union {  // (the list is in registers before any key is scored again)
    Listed listed;
    double part[SelSize<THREADS>::PARTS][THREADS == 64 ? 1 : LIST];  // 64-bit scores by 16 heads
  } u;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int t = p.t_begin + (int)blockIdx.x;
  const int k = a.topk;
  int32_t* ids = a.out + (int64_t)t * k;
  const RowPos r = locate(a, p, t);
  const int n = r.b < 0 ? 0 : r.thr;
  const int32_t* table = r.b < 0 ? nullptr : a.block_table + (int64_t)r.b * a.table_len;
  float* g = p.score + (int64_t)(t - p.t_begin) * p.width;

  if (n <= k) {  // every row there is
    int at = 0;
    for (int j0 = 0; j0 < n; j0 += THREADS) {
      const int j = j0 + tid;
      bool there = false;
      if (j < n) {
        const int page = table[p.page_div.div(j)];
        there = page >= 0 && page < a.block_num;
      }
      int all;
      const int pos = at + block_before<THREADS>(there, SLOT_IDS, sh, all);
      if (there) ids[pos] = j;
      at += all;
      __syncthreads();
    }
    for (int i = at + tid; i < k; i += THREADS) ids[i] = -1;
    return;
  }

  float err = 0.0f;  // the bound on a score's error
  auto from_registers = [&]() -> bool {
    float x[VPT];
    int id[SAMPLED ? VPT : 1];
    const bool listed = SAMPLED && n > CAP;
    auto none = [] { return make_float4(SEL_NONE, SEL_NONE, SEL_NONE, SEL_NONE); };
    auto load4 = [&](int j) {
      float4 v = none();
      if (j < n) v = *(const float4*)(g + j);
      if (j + 1 >= n) v.y = SEL_NONE;
      if (j + 2 >= n) v.z = SEL_NONE;
      if (j + 3 >= n) v.w = SEL_NONE;
      return v;
    };
    const int runs = (n + 4 * THREADS - 1) / (4 * THREADS);  // of !listed values
    float4 sample = none();
    if (listed) {
      sample = *(const float4*)(g + 4 * (int)((int64_t)tid * (n / 4) / THREADS));
    } else {
#pragma unroll
      for (int i = 0; i < VPT; i += 4) {
        const float4 v = i / 4 < runs ? load4(i * THREADS + 4 * tid) : none();
        x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
      }
    }
    float kn = 0.0f;
    {
      const SelSplit sp = r.rows < p.few_rows ? p.few : p.many;
      const int thr_end = thr_at(a, p, min(r.last, p.t_end) - 1), keys = piece_keys(sp, thr_end);
      const int parts = (thr_end + keys - 1) / keys * sp.norms;
      const float* kp = p.k_norm + (int64_t)r.b * p.norm_stride;
      for (int i = lane; i < parts; i += 64) kn = max_nonneg(kn, kp[i]);
      kn = as_float(__builtin_amdgcn_readlane(
          wave_scan(as_int(kn), 0, [](int a, int b) { return max(a, b); }), 63));
    }
    const float wn = p.w_norm[t - p.t_begin];
    err = score_error(a, wn, kn);
    if (!(err > 0.0f) || err == __builtin_inff()) return false;
    for (int i = tid; i < BINS; i += THREADS) sh.bins[i] = 0;
    if (tid == 0) {
      sh.count = 0;
      sh.found = 0;
    }

    float floor_x = SEL_NONE;  // listed: every value at or above it is in the list
    if (listed) {
      // 4 THREADS scores in runs of four, evenly over the row; the list takes what is at or
      // above the bin of their want-th largest, a little over topk's share: 6 deviations of a
      // sample of half as many independent ones
      const float share = (float)k * (4.0f * THREADS) / (float)n;
      const int want = (int)(share + 6.0f * sqrtf(2.0f * share) + 8.0f);
      if (n > SEL_SAMPLED_KEYS || (float)want * (float)n > 0.85f * CAP * (4.0f * THREADS)) return false;
      auto low = [](float v) { return v != SEL_NONE ? v : SEL_MAX; };
      float lo = fminf(fminf(low(sample.x), low(sample.y)), fminf(low(sample.z), low(sample.w)));
      float hi = fmaxf(fmaxf(sample.x, sample.y), fmaxf(sample.z, sample.w));
      block_range<THREADS>(lo, hi, sh);
      const BinMap<THREADS> m = BinMap<THREADS>::of(lo, hi);
      if (!(lo < hi) || !m.usable()) return false;
      auto tally = [&](float v) {
        if (v != SEL_NONE) atomicAdd(&sh.bins[m.bin(v)], 1u);
      };
      tally(sample.x), tally(sample.y), tally(sample.z), tally(sample.w);
      __syncthreads();
      find_bin<THREADS>(want, SLOT_SAMPLE, sh);
      floor_x = m.edge(sh.found);
      // (the first bin also takes what the sample has missed below it)
      if (sh.found == 0) floor_x = -SEL_MAX;
      // four runs of a thread at a time, the next four on their way
      float4 y[4], z[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = load4(4 * (tid + i * THREADS));
      for (int j0 = 0; j0 < n; j0 += 16 * THREADS) {
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = load4(j0 + 16 * THREADS + 4 * (tid + i * THREADS));
        int mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mine += (y[i].x >= floor_x) + (y[i].y >= floor_x) + (y[i].z >= floor_x) + (y[i].w >= floor_x);
        const int incl = wave_incl(mine);
        int at = 0;
        if (lane == 63) at = atomicAdd(&sh.count, incl);
        at = __builtin_amdgcn_readlane(at, 63) + incl - mine;
        auto add = [&](float v, int j) {
          if (v >= floor_x) {
            if (at < CAP) {
              u.listed.x[at] = v;
              u.listed.id[at] = j;
            }
            ++at;
          }
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = j0 + 4 * (tid + i * THREADS);
          add(y[i].x, j);
          add(y[i].y, j + 1);
          add(y[i].z, j + 2);
          add(y[i].w, j + 3);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = z[i];
      }
      for (int i = tid; i < (n + 31) / 32; i += THREADS) map[i] = 0;
      for (int i = tid; i < BINS; i += THREADS) sh.bins[i] = 0;
      __syncthreads();
      const int all = sh.count;
      if (all > CAP || all < k) return false;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e = tid + i * THREADS;
        x[i] = e < all ? u.listed.x[e] : SEL_NONE;
        if (SAMPLED) id[i] = e < all ? u.listed.id[e] : 0;
      }
    }
    auto id_of = [&](int i) { return listed ? id[SAMPLED ? i : 0] : (i >> 2) * 4 * THREADS + 4 * tid + (i & 3); };
    auto take = [&](int j) {
      if (listed) {
        atomicOr(&map[j >> 5], 1u << (j & 31));
      } else {
        atomicOr(&map[(j >> 8) * 8 + (j & 3) * 2 + ((j >> 7) & 1)], 1u << ((j >> 2) & 31));
      }
    };
    // the votes of a wave's four values i..i + 3
    auto put_votes = [&](int i, uint64_t m0, uint64_t m1, uint64_t m2, uint64_t m3) {
      const uint64_t m = lane == 0 ? m0 : lane == 1 ? m1 : lane == 2 ? m2 : m3;
      if (lane < 4) ((uint64_t*)map)[((i >> 2) * WAVES + wave) * 4 + lane] = m;
    };

    // the range, and how many rows there are to choose from
    float lo = SEL_MAX, hi = -SEL_MAX;
    int there = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const bool is = x[i] != SEL_NONE;
      lo = fminf(lo, is ? x[i] : SEL_MAX);
      hi = fmaxf(hi, x[i]);
      there += is;
    }
    block_range<THREADS>(lo, hi, sh);  // (a barrier: the list's length has been read)
    if (tid == 0) sh.count = 0;
    there = block_sum<THREADS>(there, SLOT_THERE, sh);
    if (there > 0 && (lo <= -SEL_MAX || hi >= SEL_MAX)) {  // a score left fp32's range
      err = __builtin_inff();
      return false;
    }
    if (there <= k) {
#pragma unroll
      for (int i = 0; i < VPT; i += 4) {
        if (!listed && i / 4 < runs) {
          put_votes(i, __ballot(x[i] != SEL_NONE), __ballot(x[i + 1] != SEL_NONE),
                    __ballot(x[i + 2] != SEL_NONE), __ballot(x[i + 3] != SEL_NONE));
        }
      }
      if (listed) return false;  // (it has topk values or more)
    } else {
      // 1. [e_lo, e_hi] around the topk-th largest, wide enough for the bound on both sides:
      // bins over the range, and over one bin's range where that holds too many
      int need = k, bin;
      BinMap<THREADS> m;
      for (int round = 0;; ++round) {
        m = BinMap<THREADS>::of(lo, hi);
        if (!(lo < hi) || !m.usable() || round == 4) return false;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          if (x[i] >= lo && x[i] <= hi) atomicAdd(&sh.bins[m.bin(x[i])], 1u);
        }
        __syncthreads();
        find_bin<THREADS>(need, SLOT_COUNT, sh);
        bin = sh.found;
        need -= sh.below;
        if (sh.in_bin <= LIST / 2) break;
        float l2 = SEL_MAX, h2 = -SEL_MAX;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          if (x[i] >= lo && x[i] <= hi && m.bin(x[i]) == bin) l2 = fminf(l2, x[i]), h2 = fmaxf(h2, x[i]);
        }
        block_range<THREADS>(l2, h2, sh);
        lo = l2;
        hi = h2;
        for (int i = tid; i < BINS; i += THREADS) sh.bins[i] = 0;
        __syncthreads();
      }
      const float slop = 2.0f * err + 4e-6f * (fabsf(lo) + fabsf(hi));
      const float e_lo = m.edge(bin) - slop, e_hi = m.edge(bin + 1) + slop;
      if (!(e_lo > -SEL_MAX) || !(e_hi < SEL_MAX) || (listed && e_lo < floor_x)) return false;

      // 2. values above are taken, those inside are listed
      int above = 0;
      auto classify = [&](int i) -> uint64_t {
        const bool over = x[i] > e_hi;
        const uint64_t vote = __ballot(over);
        above += (int)__popcll(vote);
        if (listed && over) take(id_of(i));
        if (!over && x[i] >= e_lo) {
          const int e = atomicAdd(&sh.count, 1);
          if (e < LIST) {
            sh.list_x[e] = x[i];
            sh.list_j[e] = id_of(i);
          }
        }
        return vote;
      };
#pragma unroll
      for (int i = 0; i < VPT; i += 4) {
        if (!listed && i / 4 >= runs) continue;
        const uint64_t v0 = classify(i), v1 = classify(i + 1), v2 = classify(i + 2), v3 = classify(i + 3);
        if (!listed) put_votes(i, v0, v1, v2, v3);
      }
      above = block_sum<THREADS>(lane == 0 ? above : 0, SLOT_ABOVE, sh);
      __syncthreads();
      const int inside = sh.count;
      need = k - above;
      if (inside > LIST || need < 1 || need > inside) return false;
      if (tid == 0) sh.close = sh.sure = 0;
      rank_list<THREADS>(inside, sh.list_x, sh.list_j, [&](int i, int rank) {
        if (rank == need - 1) sh.value = sh.list_x[i];
      });
      __syncthreads();
      const float kth = sh.value, b_lo = kth - 2.0f * err, b_hi = kth + 2.0f * err;
      if (b_lo < e_lo || b_hi > e_hi) return false;
      for (int i = tid; i < inside; i += THREADS) {
        const float y = sh.list_x[i];
        if (y > b_hi) {
          take(sh.list_j[i]);
          atomicAdd(&sh.sure, 1);
        } else if (y >= b_lo) {
          sh.close_j[atomicAdd(&sh.close, 1)] = sh.list_j[i];
        }
      }
      __syncthreads();
      const int close = sh.close, rest = need - sh.sure;  // `rest` of the `close` rows are taken
      if (close == rest) {
        for (int i = tid; i < close; i += THREADS) take(sh.close_j[i]);
      } else {
        const int groups = (close + 15) / 16, heads16 = (a.heads + 15) / 16;
        if (WAVES == 1) {
          for (int i = 0; i < close; i += 16) {
            const uint64_t key = order64<T, FP8>(a, p, t, table, sh.close_j[min(i + (lane & 15), close - 1)], lane);
            if (lane < 16 && i + lane < close) sh.list_key[i + lane] = key;
          }
        } else {
          for (int i = wave; i < groups * heads16; i += WAVES) {
            const int e = i / heads16 * 16, h16 = i % heads16;
            const double s = score64_part<T, FP8>(a, p, t, table, sh.close_j[min(e + (lane & 15), close - 1)],
                                                  16 * h16, lane);
            if (lane < 16 && e + lane < close) u.part[h16][e + lane] = s;
          }
          __syncthreads();
          for (int i = tid; i < close; i += THREADS) {
            double s = 0.0;
            for (int h16 = 0; h16 < heads16; ++h16) s += u.part[h16][i];
            sh.list_key[i] = order_of(s * key_scale64<FP8>(a, p, table, sh.close_j[i]));
          }
        }
        __syncthreads();
        rank_list<THREADS>(close, sh.list_key, sh.close_j, [&](int i, int rank) {
          if (rank < rest) take(sh.close_j[i]);
        });
      }
    }
    __syncthreads();

    // 3. the ids in order
    const int words = listed ? (n + 31) / 32 : (n + 255) / 256 * 8;
    const int per = (words + THREADS - 1) / THREADS, w0 = min(tid * per, words), w1 = min(w0 + per, words);
    auto word = [&](int w) -> uint32_t {
      if (listed) return map[w];
      const unsigned char* votes = (const unsigned char*)map + (w >> 3) * 32 + (w & 7);
      return every_fourth(votes[0]) | every_fourth(votes[8]) << 1 | every_fourth(votes[16]) << 2 |
             every_fourth(votes[24]) << 3;
    };
    int mine = 0, all;
    for (int w = w0; w < w1; ++w) mine += __popc(word(w));
    int pos = block_before<THREADS>(mine, SLOT_IDS, sh, all);
    for (int w = w0; w < w1; ++w) {
      for (uint32_t bits = word(w); bits; bits &= bits - 1) ids[pos++] = 32 * w + __builtin_ctz(bits);
    }
    for (int i = all + tid; i < k; i += THREADS) ids[i] = -1;
    return true;
  };
  if (!from_registers()) {
    __syncthreads();
    select_from_memory<T, FP8, THREADS>(a, p, t, n, err, g, table, sh);
  }
}

// ---------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------

// Scores of a pass may take this much of the workspace; more query rows take more passes.
constexpr int64_t SEL_PASS_BYTES = 512ll << 20;

struct PassPlan {
  SelPlan p;
  int rows;            // query rows of a pass
  int64_t bytes;       // workspace
};

PassPlan plan_passes(const SasSelectArgs& a) {
  PassPlan r;
  SelPlan& p = r.p;
  const int keys = a.max_keys < 1 ? 1 : a.max_keys;
  p.width = (keys + 31) / 32 * 32;
  int64_t rows = SEL_PASS_BYTES / ((int64_t)p.width * 4);
  rows = rows < 8 ? 8 : rows / 8 * 8;
  r.rows = (int)(rows < a.tokens ? rows : a.tokens);
  const int64_t per_seq = a.batch > 0 ? (int64_t)a.tokens / a.batch : 0;
  // From four query rows a sequence on, keys shared through LDS beat a row on its own (32
  // sequences of 16384 keys, 4 rows: 71 us against 81; at 2 rows the shared kernel has six of
  // its eight waves idle: 13 sequences, 36 us against 21). Where the rows differ by sequence, as
  // the device alone knows, both kernels are launched and each sequence has one of them: tiles of
  // eight single rows would take their sequences in turn (a step of 633 rows in 23 sequences, 16
  // of one row: 54 us by tiles alone, 32 + 8 us by both kernels).
  const bool even = a.rows_per_seq > 0 && !a.cu_seqlens_q;
  p.few_rows = even ? (a.rows_per_seq < SEL_FEW_ROWS ? INT32_MAX : 0)
                    : a.batch == 1 ? (a.tokens < SEL_FEW_ROWS ? INT32_MAX : 0)
                                   : per_seq <= 2 ? INT32_MAX : SEL_FEW_ROWS;
  // Enough workgroups to fill the chip, of at least 64 keys a slice. Decode rows, 1024 / 2048
  // workgroups: even lengths (64 x 32768 keys) 110 / 118 us, uneven ones (128 x 32768 to 131072,
  // fp8) 383 / 357 us; even batches are the ones that lose least. Tiles of eight rows, 256 / 512 /
  // 1024: a mixed step of 633 rows 27 / 33 / 41 us, 1024 rows over 4096 keys 81 / 85 / 98 us, 2048
  // rows of 128 heads over 8192 keys 733 / 660 / 691 us.
  auto split = [&](int64_t groups, int64_t wanted, int slices, int norms) {
    const int64_t most = (p.width + 64 * slices - 1) / (64 * slices);
    const int64_t pieces = (wanted + groups - 1) / (groups < 1 ? 1 : groups);
    return SelSplit{(int)(pieces < 1 ? 1 : pieces > most ? most : pieces), slices, norms};
  };
  p.few = split(p.few_rows == SEL_FEW_ROWS ? a.batch : r.rows, 2048, STREAM_WAVES, STREAM_WAVES);
  p.many = split((r.rows + TILE_WAVES - 1) / TILE_WAVES, 256, 1, TILE_WAVES);
  const int few_norms = p.few.chunks * p.few.norms, many_norms = p.many.chunks * p.many.norms;
  p.norm_stride = few_norms > many_norms ? few_norms : many_norms;
  // every part starts on 16 bytes
  const int64_t w_floats = ((int64_t)r.rows + 3) / 4 * 4;
  const int64_t k_floats = ((int64_t)a.batch * p.norm_stride + 3) / 4 * 4;
  r.bytes = 4 * (w_floats + k_floats + (int64_t)r.rows * p.width);
  p.w_norm = (float*)a.workspace;
  p.k_norm = p.w_norm + w_floats;
  p.score = p.k_norm + k_floats;
  p.page_div = FastDiv::of(a.block_size);
  p.ratio_div = FastDiv::of(a.cmp_ratio);
  return r;
}

int check_select(const SasSelectArgs* a) {
  auto fail = [&](const char* what, int rc = SAS_E_INVALID) {
    set_error(std::string("sas_topk_select: ") + what);
    return rc;
  };
  if (!a) return fail("null arguments");
  if (a->batch < 0 || a->tokens < 0 || a->rows_per_seq < 0) return fail("negative size");
  if (a->heads < 1 || a->heads > SAS_SELECT_MAX_HEADS) return fail("heads must be 1 to 128");
  if (a->dim != 64 && a->dim != 128) return fail("dim must be 64 or 128", SAS_E_UNSUPPORTED);
  if (a->topk < 1) return fail("topk must be at least 1");
  if (a->cmp_ratio < 1) return fail("cmp_ratio must be at least 1");
  if (a->dtype != SAS_DTYPE_BF16 && a->dtype != SAS_DTYPE_FP16) return fail("dtype");
  if (a->key_format != SAS_ROW_NATIVE && a->key_format != SAS_ROW_FP8_INDEX) return fail("key_format");
  if (a->block_num < 1 || a->block_size < 1 || a->table_len < 1) return fail("bad cache geometry");
  if ((int64_t)a->block_num * a->block_size >= (1ll << 31)) {
    return fail("2^31 cache rows or more", SAS_E_UNSUPPORTED);
  }
  if (a->max_keys < 1 || a->max_keys > (int64_t)a->table_len * a->block_size ||
      a->max_keys > SAS_SELECT_MAX_KEYS) {
    return fail("max_keys must be at least 1, and within the block table and SAS_SELECT_MAX_KEYS");
  }
  if ((int64_t)a->block_num * a->block_size * (a->key_format == SAS_ROW_FP8_INDEX ? a->dim + 4 : 2 * a->dim) >=
      (1ll << 36)) {
    return fail("an index cache of 64 GiB or more", SAS_E_UNSUPPORTED);
  }
  if (a->key_format == SAS_ROW_FP8_INDEX && (int64_t)a->block_size * (a->dim + 4) % 16) {
    return fail("fp8 index pages must be a multiple of 16 bytes");
  }
  if (a->rows_per_seq > 0 && (int64_t)a->rows_per_seq * a->batch != a->tokens) {
    return fail("tokens must be batch * rows_per_seq");
  }
  return SAS_OK;
}

template <typename T, bool FP8, int D, int MT>
void launch_scores(const SasSelectArgs& a, const SelPlan& p, hipStream_t st) {
  const int64_t rows = p.t_end - p.t_begin, tiles = (rows + TILE_WAVES - 1) / TILE_WAVES;
  if (p.few_rows < INT32_MAX) {
    hipLaunchKernelGGL((score_tile_kernel<T, FP8, D, MT>), dim3((unsigned)(tiles * p.many.chunks)),
                       dim3(64 * TILE_WAVES), 0, st, a, p);
  }
  if (p.few_rows > 0) {
    const int64_t alone = p.few_rows == SEL_FEW_ROWS ? (int64_t)a.batch * (SEL_FEW_ROWS - 1) : rows;
    hipLaunchKernelGGL((score_stream_kernel<T, FP8, D, MT>), dim3((unsigned)(alone * p.few.chunks)),
                       dim3(64 * STREAM_WAVES), 0, st, a, p);
  }
}

template <typename T, bool FP8>
void launch_pass(const SasSelectArgs& a, const SelPlan& p, hipStream_t st) {
  if (a.max_keys > a.topk) {  // else every row takes all it may see: no scores
    const int mt = (a.heads + 31) / 32;
    if (a.dim == 128) {
      if (mt == 1) launch_scores<T, FP8, 128, 1>(a, p, st);
      else if (mt == 2) launch_scores<T, FP8, 128, 2>(a, p, st);
      else launch_scores<T, FP8, 128, 4>(a, p, st);
    } else {
      if (mt == 1) launch_scores<T, FP8, 64, 1>(a, p, st);
      else if (mt == 2) launch_scores<T, FP8, 64, 2>(a, p, st);
      else launch_scores<T, FP8, 64, 4>(a, p, st);
    }
  }
  const int rows = p.t_end - p.t_begin;
  const dim3 grid((unsigned)rows);
  // The workgroup of a row. Of many short rows one wave each: 1024 / 1536 / 2048 / 3000 / 6771 rows
  // of up to 2048 scores take 33 / 33 / 40 / 45 / 71 us with 64 threads and 22 / 34 / 39 / 54 /
  // 106 us with 256. Up to 8192 scores 256 threads hold a row (32 rows of 4096: 15.4 us, with 1024
  // threads 17.1); longer rows are sampled first (64 rows of 32768: 32.1 us, all of a row in the
  // registers of 1024 threads 34.1).
  if (a.max_keys <= 2048 && rows >= 2048) {
    hipLaunchKernelGGL((select_kernel<T, FP8, 64, 32, false>), grid, dim3(64), 0, st, a, p);
  } else if (a.max_keys <= 8192) {
    hipLaunchKernelGGL((select_kernel<T, FP8, 256, 32, false>), grid, dim3(256), 0, st, a, p);
  } else {
    hipLaunchKernelGGL((select_kernel<T, FP8, 1024, 8, true>), grid, dim3(1024), 0, st, a, p);
  }
}

}  // namespace
}  // namespace sas

extern "C" int64_t sas_topk_select_workspace(const SasSelectArgs* a) {
  if (sas::check_select(a) != SAS_OK) return -1;
  return sas::plan_passes(*a).bytes;
}

extern "C" int sas_topk_select(const SasSelectArgs* a, void* stream) {
  const int rc = sas::check_select(a);
  if (rc != SAS_OK || a->tokens == 0) return rc;
  auto fail = [&](const char* what) {
    sas::set_error(std::string("sas_topk_select: ") + what);
    return (int)SAS_E_INVALID;
  };
  if (!a->q || !a->weights || !a->keys || !a->block_table || !a->seqused_kv || !a->out ||
      !a->workspace || (a->rows_per_seq == 0 && !a->cu_seqlens_q)) {
    return fail("null pointer");
  }
  if (((uintptr_t)a->q | (uintptr_t)a->keys | (uintptr_t)a->workspace) & 15) {
    return fail("q, keys and workspace must be aligned to 16 bytes");
  }
  const sas::PassPlan r = sas::plan_passes(*a);
  if (a->workspace_bytes < r.bytes) {
    sas::set_error("sas_topk_select: workspace smaller than sas_topk_select_workspace");
    return SAS_E_CAPACITY;
  }
  const hipStream_t st = (hipStream_t)stream;
  for (int t = 0; t < a->tokens; t += r.rows) {
    sas::SelPlan p = r.p;
    p.t_begin = t;
    p.t_end = (int64_t)t + r.rows < a->tokens ? t + r.rows : a->tokens;
    const bool fp8 = a->key_format == SAS_ROW_FP8_INDEX;
    if (a->dtype == SAS_DTYPE_BF16) {
      fp8 ? sas::launch_pass<__bf16, true>(*a, p, st) : sas::launch_pass<__bf16, false>(*a, p, st);
    } else {
      fp8 ? sas::launch_pass<_Float16, true>(*a, p, st)
          : sas::launch_pass<_Float16, false>(*a, p, st);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
      sas::set_error(std::string("sas_topk_select: ") + hipGetErrorString(e));
      return SAS_E_HIP;
    }
  }
  return SAS_OK;
}

extern "C" int sas_select_args_struct_size(void) { return (int)sizeof(SasSelectArgs); }
