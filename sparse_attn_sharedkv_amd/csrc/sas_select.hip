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
// most E = c W K, c = (D + H + 4) 2^-23, W = sum_h |w_h| |q_h|, K = max_j |k_j| (below), so a row
// whose fp32 score is more than 2 E above the topk-th largest fp32 score is in, one more than 2 E
// below it is out, and the few in between are scored again in 64 bits. Ids are therefore those
// of 64-bit scores for any split of the work, any batch and any tile.
//
// The bound. Products of two 16-bit numbers are exact in fp32. A dot product's D terms are added
// in some order and with some grouping inside the matrix instruction; each addition loses at most
// 2^-23 of the sum of the magnitudes (a rounding 2^-24, a truncated alignment twice that), so it
// is off by at most D 2^-23 sum |q_i k_i| <= D 2^-23 |q| |k|. max(0, x) moves no two values
// further apart. The weighted sum of H terms rounds at most H + 2 times (2^-24 each, of a sum of
// magnitudes below (1 + small) W K), an fp8 row's scale once more. c has the rest as slack for
// terms of second order and for the norms' own rounding. 2^-50 is added to each norm for products
// below fp32's normal range. A bound that is not finite (infinities, NaN, norms beyond fp32)
// has the whole row scored in 64 bits.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/sas_mi355x.h"
#include "sas_items.h"

namespace sas {

void set_error(const std::string& msg);

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
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
  static __device__ float lo(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[0]; }
  static __device__ float hi(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[1]; }
};

// Eight e4m3 codes as eight elements of T (exact: e4m3 fits in both 16-bit types).
template <typename T>
__device__ inline u32x4 widen_e4m3(u32x2 c) {
  typename Elem<T>::v8 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(c[i], false);
    const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(c[i], true);
    r[4 * i] = (T)a[0], r[4 * i + 1] = (T)a[1], r[4 * i + 2] = (T)b[0], r[4 * i + 3] = (T)b[1];
  }
  return __builtin_bit_cast(u32x4, r);
}

// What both kernels know of a launch besides its arguments.
struct SelPlan {
  int t_begin, t_end;   // query rows of this pass
  int width;            // scores kept for a row (row stride of the workspace)
  int chunk, chunks;    // keys of a workgroup, and such pieces in `width`
  int slices;           // waves that share a chunk's keys (each leaves its own key norm)
  int wq;               // query rows of a workgroup
  FastDiv page_div, ratio_div;
  float* w_norm;        // [rows of the pass] W of each row
  float* k_norm;        // [batch][chunks][slices] largest |k|^2 of the keys seen
  float* score;         // [rows of the pass][width]
};

struct RowPos {
  int b;     // sequence, -1: a row of no sequence
  int thr;   // keys the row may choose from
  int last;  // first query row behind the sequence's (or behind the run of rows of no sequence)
};

__device__ inline RowPos locate(const SasSelectArgs& a, const SelPlan& p, int t) {
  RowPos r;
  int s, act_q;
  if (a.rows_per_seq > 0) {
    const int b = t / a.rows_per_seq;
    s = t - b * a.rows_per_seq;
    act_q = a.cu_seqlens_q ? a.cu_seqlens_q[b + 1] - a.cu_seqlens_q[b] : a.rows_per_seq;
    if (act_q > a.rows_per_seq) act_q = a.rows_per_seq;
    if (s >= act_q) return {-1, 0, (b + 1) * a.rows_per_seq};
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
    if (lo < 0) return {-1, 0, a.batch > 0 ? a.cu_seqlens_q[0] : a.tokens};
    const int first = a.cu_seqlens_q[lo], end = a.cu_seqlens_q[lo + 1];
    if (t >= end) return {-1, 0, lo + 1 < a.batch ? a.cu_seqlens_q[lo + 1] : a.tokens};
    r.b = lo;
    s = t - first;
    act_q = end - first;
    r.last = end;
  }
  const ItemGeom g = item_geom_div(act_q, a.seqused_kv[r.b], s, -1, 2, p.ratio_div, 0);
  r.thr = min(g.thr, a.max_keys);
  return r;
}

// thr of the last row before `end` that belongs to the same sequence as a row with `thr` at `t`.
__device__ inline int thr_at(const SasSelectArgs& a, const SelPlan& p, int t) {
  return locate(a, p, t).thr;
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

__device__ inline int frag_dim(int p, int u, int hf) { return 32 * p + 16 * hf + 8 * u; }

template <typename T, int D, int MT>
struct QueryFrags {
  u32x4 q[MT][D / 16];
  f32x16 w[MT];

  __device__ void load(const SasSelectArgs& a, int t, int lane) {
    const int m = lane & 31, hf = lane >> 5;
    const T* base = (const T*)a.q + (int64_t)t * a.heads * D;
    const float* wb = a.weights + (int64_t)t * a.heads;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int h = 32 * mt + m;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        q[mt][k] = h < a.heads ? *(const u32x4*)(base + (int64_t)h * D + frag_dim(k >> 1, k & 1, hf))
                               : u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int hh = 32 * mt + 8 * (i >> 2) + 4 * hf + (i & 3);
        w[mt][i] = hh < a.heads ? wb[hh] : 0.0f;
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
      if (h < a.heads) s += fabsf(a.weights[(int64_t)t * a.heads + h]) * (sqrtf(n2) + SEL_TINY);
    }
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) s += __shfl_xor(s, off, 64);
    return s;
  }

  // the score of key lane & 31 without its scale
  __device__ float score(const u32x4 k[D / 16]) const {
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      f32x16 acc = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) acc = Elem<T>::mfma(q[mt][kk], k[kk], acc);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i & 3] = fmaf(fmaxf(acc[i], 0.0f), w[mt][i], s[i & 3]);
    }
    const float r = (s[0] + s[1]) + (s[2] + s[3]);
    return r + __shfl_xor(r, 32, 64);
  }
};

template <typename T, int D>
__device__ inline float key_norm2(const u32x4 k[D / 16]) {
  float n = 0.0f;
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
    for (int e = 0; e < 4; ++e) n = Elem<T>::dot2(k[kk][e], n);
  return n + __shfl_xor(n, 32, 64);
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

// Decode: few query rows a sequence. A workgroup's four waves take wq query rows times 4 / wq
// slices of a chunk's keys; nothing is shared and there is no barrier. Keys go from memory to
// registers, the next tile's in flight under the current one's products. Bound by the keys'
// bytes: a key row is read once for each query row.
template <typename T, bool FP8, int D, int MT>
__global__ __launch_bounds__(256) void score_stream_kernel(SasSelectArgs a, SelPlan p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 31, hf = lane >> 5;
  const int piece = (int)(blockIdx.x % (unsigned)p.chunks);
  const int t = p.t_begin + (int)(blockIdx.x / (unsigned)p.chunks) * p.wq + wave % p.wq;
  if (t >= p.t_end) return;
  const RowPos r = locate(a, p, t);
  const int lo = piece * p.chunk;
  if (r.b < 0 || r.thr <= a.topk || lo >= r.thr) return;
  const int hi = min(lo + p.chunk, r.thr), slice = wave / p.wq, step = 32 * p.slices;

  QueryFrags<T, D, MT> qf;
  qf.load(a, t, lane);
  if (piece == 0 && slice == 0) {
    const float w = qf.bound(a, t, lane);
    if (lane == 0) p.w_norm[t - p.t_begin] = w;
  }
  const bool norms = t == min(r.last, p.t_end) - 1;
  float kn = 0.0f;
  const int32_t* table = a.block_table + (int64_t)r.b * a.table_len;
  float* out = p.score + (int64_t)(t - p.t_begin) * p.width;

  auto page_of = [&](int j) { return j < hi ? table[p.page_div.div(j)] : -1; };
  auto load = [&](int j, int page, u32x4 k[D / 16], float& scale) {
    const bool ok = page >= 0 && page < a.block_num;
    const int at = j - p.page_div.div(j) * a.block_size;
    if (!FP8) {
      const T* row = (const T*)a.keys + (ok ? (int64_t)page * a.block_size + at : 0) * D;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) k[kk] = *(const u32x4*)(row + frag_dim(kk >> 1, kk & 1, hf));
    } else {
      const unsigned char* pg = (const unsigned char*)a.keys +
                                (ok ? (int64_t)page : 0) * a.block_size * (D + 4);
      const unsigned char* row = pg + (ok ? at : 0) * D;
#pragma unroll
      for (int q = 0; q < D / 32; ++q) k[q] = *(const u32x4*)(row + 32 * q + 16 * hf);
      scale = *(const float*)(pg + (int64_t)a.block_size * D + 4 * (ok ? at : 0));
    }
    return ok;
  };

  int j = lo + 32 * slice + n;
  int page_next = page_of(j + step);
  u32x4 cur[D / 16], nxt[D / 16];
  float sc_cur = 1.0f, sc_nxt = 1.0f;
  bool ok_cur = load(j, page_of(j), cur, sc_cur), ok_nxt = false;
  for (int base = lo + 32 * slice; base < hi; base += step, j += step) {
    const int page_far = page_of(j + 2 * step);
    ok_nxt = load(j + step, page_next, nxt, sc_nxt);
    page_next = page_far;
    u32x4 k[D / 16];
    if (FP8) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const u32x4 c = cur[kk >> 1];
        k[kk] = widen_e4m3<T>(kk & 1 ? u32x2{c[2], c[3]} : u32x2{c[0], c[1]});
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) k[kk] = cur[kk];
    }
    if (norms) {
      float n2 = key_norm2<T, D>(k);
      if (FP8) n2 *= sc_cur * sc_cur;
      if (ok_cur) kn = max_nonneg(kn, n2);
    }
    float s = qf.score(k);
    if (FP8) s *= sc_cur;
    if (hf == 0 && j < hi) out[j] = ok_cur ? kept_score(s) : SEL_NONE;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) cur[kk] = nxt[kk];
    sc_cur = sc_nxt;
    ok_cur = ok_nxt;
  }
  if (norms) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) kn = max_nonneg(kn, __shfl_xor(kn, off, 64));
    if (lane == 0) p.k_norm[((int64_t)r.b * p.chunks + piece) * p.slices + slice] = kn;
  }
}

// Prefill: many query rows a sequence. A workgroup's eight waves own one query row each and
// share the keys, 64 at a time through LDS (two stages, the next one's loads in flight under the
// current one's products; fp8 codes are widened on the way in). Bound by the matrix cores.
// A tile of eight rows that spans sequences takes them one after the other.
constexpr int TILE_WAVES = 8;
constexpr int TILE_KEYS = 64;

// byte offset of 16-byte chunk c of row r in a stage: the rows' chunks are rotated against each
// other so that 16 lanes reading one chunk of 16 rows touch every bank once
template <int D>
__device__ inline int stage_at(int r, int c) {
  return D == 128 ? r * 256 + ((c ^ (r & 15)) << 4) : r * 128 + ((c ^ ((r >> 1) & 7)) << 4);
}

template <typename T, bool FP8, int D, int MT>
__global__ __launch_bounds__(64 * TILE_WAVES) void score_tile_kernel(SasSelectArgs a, SelPlan p) {
  __shared__ __attribute__((aligned(256))) unsigned char stage[2][TILE_KEYS * D * 2];
  __shared__ float key_scale[2][TILE_KEYS];
  __shared__ int key_ok[2][TILE_KEYS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 31, hf = lane >> 5;
  const int piece = (int)(blockIdx.x % (unsigned)p.chunks);
  const int tiles = (p.t_end - p.t_begin + TILE_WAVES - 1) / TILE_WAVES;
  // the last rows of a causal prefill have the most keys: they start first
  const int t0 = p.t_begin + (tiles - 1 - (int)(blockIdx.x / (unsigned)p.chunks)) * TILE_WAVES;
  const int t1 = min(t0 + TILE_WAVES, p.t_end), t = t0 + wave;
  const int lo = piece * p.chunk;
  // the thread's part of a stage: bytes [32 part, +32) of native row `row`, or 16 codes
  constexpr int PARTS = 64 * TILE_WAVES / TILE_KEYS;   // 8 threads a row
  constexpr int LOADS = FP8 ? 1 : D * 2 / (16 * PARTS);  // 16-byte loads of a thread
  const int row = threadIdx.x / PARTS, part = threadIdx.x % PARTS;
  const bool loads_codes = !FP8 || part < D / 16;

  QueryFrags<T, D, MT> qf;
  for (int ts = t0; ts < t1;) {
    const RowPos seg = locate(a, p, ts);
    const int te = max(min(seg.last, t1), ts + 1);
    const int thr_end = seg.b < 0 ? 0 : thr_at(a, p, te - 1);
    const int hi = min(lo + p.chunk, thr_end);
    if (thr_end <= a.topk || lo >= thr_end) {
      ts = te;
      continue;
    }
    const bool mine = t >= ts && t < te;
    const int my_thr = mine ? thr_at(a, p, t) : 0;
    const bool active = mine && my_thr > a.topk && lo < my_thr;
    const bool norms = mine && t == min(seg.last, p.t_end) - 1;
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

    u32x4 held[LOADS];
    float held_scale = 1.0f;
    int held_ok = 0;
    auto page_of = [&](int j) { return j < hi ? table[p.page_div.div(j)] : -1; };
    auto fetch = [&](int j, int page) {
      held_ok = page >= 0 && page < a.block_num;
      const int at = held_ok ? j - p.page_div.div(j) * a.block_size : 0;
      const int64_t pg = held_ok ? page : 0;
      if (!FP8) {
        const unsigned char* src = (const unsigned char*)a.keys + (pg * a.block_size + at) * (2 * D);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) held[i] = *(const u32x4*)(src + 16 * (part * LOADS + i));
      } else {
        const unsigned char* src = (const unsigned char*)a.keys + pg * a.block_size * (D + 4);
        if (loads_codes) held[0] = *(const u32x4*)(src + at * D + 16 * part);
        held_scale = *(const float*)(src + (int64_t)a.block_size * D + 4 * at);
      }
    };
    auto put = [&](int buf) {
      if (!FP8) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
          *(u32x4*)(stage[buf] + stage_at<D>(row, part * LOADS + i)) = held[i];
      } else if (loads_codes) {
        *(u32x4*)(stage[buf] + stage_at<D>(row, 2 * part)) =
            widen_e4m3<T>(u32x2{held[0][0], held[0][1]});
        *(u32x4*)(stage[buf] + stage_at<D>(row, 2 * part + 1)) =
            widen_e4m3<T>(u32x2{held[0][2], held[0][3]});
      }
      if (part == 0) {
        key_ok[buf][row] = held_ok;
        key_scale[buf][row] = held_scale;
      }
    };

    int page_next = page_of(lo + TILE_KEYS + row);
    fetch(lo + row, page_of(lo + row));
    put(0);
    __syncthreads();
    int buf = 0;
    for (int base = lo; base < hi; base += TILE_KEYS, buf ^= 1) {
      const bool more = base + TILE_KEYS < hi;
      if (more) {
        fetch(base + TILE_KEYS + row, page_next);
        page_next = page_of(base + 2 * TILE_KEYS + row);
      }
      if (active) {
#pragma unroll
        for (int kt = 0; kt < TILE_KEYS / 32; ++kt) {
          if (base + 32 * kt >= my_thr) break;
          const int kr = 32 * kt + n, j = base + kr;
          u32x4 k[D / 16];
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            k[kk] = *(const u32x4*)(stage[buf] + stage_at<D>(kr, frag_dim(kk >> 1, kk & 1, hf) / 8));
          const bool ok = key_ok[buf][kr];
          const float sc = FP8 ? key_scale[buf][kr] : 1.0f;
          if (norms) {
            float n2 = key_norm2<T, D>(k);
            if (FP8) n2 *= sc * sc;
            if (ok) kn = max_nonneg(kn, n2);
          }
          float s = qf.score(k);
          if (FP8) s *= sc;
          if (hf == 0 && j < my_thr && j < hi) out[j] = ok ? kept_score(s) : SEL_NONE;
        }
      }
      if (more) put(buf ^ 1);
      __syncthreads();
    }
    if (norms) {
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) kn = max_nonneg(kn, __shfl_xor(kn, off, 64));
      if (lane == 0) p.k_norm[(int64_t)seg.b * p.chunks + piece] = kn;
    }
    ts = te;
  }
}

// ---------------------------------------------------------------------------
// Selection
// ---------------------------------------------------------------------------

constexpr int SEL_BINS = 2048;
constexpr int SEL_LIST = 1024;  // rows scored again, or ranked, in LDS

template <int THREADS, int ROWCAP>
struct SelShared {
  float row[ROWCAP > 0 ? ROWCAP : 1];
  uint32_t bins[SEL_BINS];
  float list_x[SEL_LIST];
  int list_j[SEL_LIST];
  uint64_t list_key[SEL_LIST];
  int wave_a[THREADS / 64], wave_b[THREADS / 64];
  float wave_lo[THREADS / 64], wave_hi[THREADS / 64];
  int count, found, below, in_bin;
  float value;
};

__device__ inline uint64_t order_of(double s) {
  // larger score, larger number; NaN as the lowest, -0 as 0
  if (!(s == s)) s = -__builtin_inf();
  s += 0.0;
  const uint64_t u = __builtin_bit_cast(uint64_t, s);
  return u >> 63 ? ~u : u | (1ull << 63);
}

// The score of key j in 64 bits, by one wave (the same in every lane): lanes are heads, and
// where there are fewer than 64 several lanes share a head's dims.
template <typename T, bool FP8>
__device__ double score64(const SasSelectArgs& a, const SelPlan& p, int t, const int32_t* table, int j,
                          int lane) {
  const int d = a.dim;
  int hp = 1;
  while (hp < a.heads && hp < 64) hp <<= 1;
  int parts = 64 / hp;
  while (parts > d / 8) parts >>= 1;
  const int dims = d / parts;  // a multiple of 8
  const int part = lane / hp;
  const int pg = p.page_div.div(j), at = j - pg * a.block_size;
  const int64_t page = table[pg];
  const T* krow = nullptr;
  const unsigned char* crow = nullptr;
  double scale = 1.0;
  if (!FP8) {
    krow = (const T*)a.keys + (page * a.block_size + at) * d;
  } else {
    const unsigned char* base = (const unsigned char*)a.keys + page * a.block_size * (d + 4);
    crow = base + (int64_t)at * d;
    scale = (double)*(const float*)(base + (int64_t)a.block_size * d + 4 * at);
  }
  double total = 0.0;
  for (int h0 = 0; h0 < a.heads; h0 += 64) {
    const int h = h0 + (lane & (hp - 1));
    const bool live = h < a.heads && part < parts;
    double acc = 0.0;
    if (live) {
      const T* q = (const T*)a.q + ((int64_t)t * a.heads + h) * d + part * dims;
      for (int e = 0; e < dims; e += 8) {
        const u32x4 qv = *(const u32x4*)(q + e);
        const u32x4 kv = FP8 ? widen_e4m3<T>(*(const u32x2*)(crow + part * dims + e))
                             : *(const u32x4*)(krow + part * dims + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc = fma((double)Elem<T>::lo(qv[i]), (double)Elem<T>::lo(kv[i]), acc);
          acc = fma((double)Elem<T>::hi(qv[i]), (double)Elem<T>::hi(kv[i]), acc);
        }
      }
    }
    for (int off = hp; off < hp * parts; off <<= 1) acc += __shfl_xor(acc, off, 64);
    const double x = acc < 0.0 ? 0.0 : acc;  // (keeps NaN)
    double s = live && part == 0 ? x * (double)a.weights[(int64_t)t * a.heads + h] : 0.0;
    for (int off = 1; off < hp; off <<= 1) s += __shfl_xor(s, off, 64);
    total += s;
  }
  return __shfl(total * scale, 0, 64);
}

template <int THREADS>
__device__ inline int block_sum(int v, int* scratch) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  int s = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) s += scratch[i];
  return s;
}

template <typename T, bool FP8, int THREADS, int ROWCAP>
__global__ __launch_bounds__(THREADS) void select_kernel(SasSelectArgs a, SelPlan p) {
  __shared__ SelShared<THREADS, ROWCAP> sh;
  constexpr int WAVES = THREADS / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int t = p.t_begin + (int)blockIdx.x;
  const int k = a.topk;
  int32_t* ids = a.out + (int64_t)t * k;
  const RowPos r = locate(a, p, t);
  const int n = r.b < 0 ? 0 : r.thr;
  const int32_t* table = r.b < 0 ? nullptr : a.block_table + (int64_t)r.b * a.table_len;

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

  if (n <= k) {
    auto there = [&](int j) {
      const int page = table[p.page_div.div(j)];
      return page >= 0 && page < a.block_num;
    };
    emit(there, [](int) { return false; }, 0);
    return;
  }

  // the bound on a score's error
  float* g = p.score + (int64_t)(t - p.t_begin) * p.width;
  float kn = 0.0f;
  {
    const int thr_end = thr_at(a, p, min(r.last, p.t_end) - 1);
    const int parts = (thr_end + p.chunk - 1) / p.chunk * p.slices;
    const float* kp = p.k_norm + (int64_t)r.b * p.chunks * p.slices;
    for (int i = lane; i < parts; i += 64) kn = max_nonneg(kn, kp[i]);
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) kn = max_nonneg(kn, __shfl_xor(kn, off, 64));
  }
  const float wn = p.w_norm[t - p.t_begin];
  float err = (float)(a.dim + a.heads + 4) * 1.1920929e-7f * wn * (sqrtf(kn) + SEL_TINY);
  if (kn == 0.0f || wn == 0.0f) err = 0.0f;  // every score is exactly 0
  if (!(err <= SEL_MAX)) err = __builtin_inff();

  // the row into LDS where it fits, its range, and how many rows there are to choose from
  float lo = SEL_MAX, hi = -SEL_MAX;
  int there = 0, edge = 0;
  for (int j = tid; j < n; j += THREADS) {
    const float x = g[j];
    if (ROWCAP > 0) sh.row[j] = x;
    if (x != SEL_NONE) {
      lo = fminf(lo, x);
      hi = fmaxf(hi, x);
      ++there;
      edge |= fabsf(x) >= SEL_MAX;
    }
  }
  float* x_of = ROWCAP > 0 ? sh.row : g;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    lo = fminf(lo, __shfl_xor(lo, off, 64));
    hi = fmaxf(hi, __shfl_xor(hi, off, 64));
  }
  if (lane == 0) {
    sh.wave_lo[wave] = lo;
    sh.wave_hi[wave] = hi;
  }
  there = block_sum<THREADS>(there, sh.wave_a);
  edge = block_sum<THREADS>(edge, sh.wave_b);
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    lo = fminf(lo, sh.wave_lo[w]);
    hi = fmaxf(hi, sh.wave_hi[w]);
  }
  if (edge) err = __builtin_inff();
  if (there <= k) {
    emit([&](int j) { return x_of[j] != SEL_NONE; }, [](int) { return false; }, 0);
    return;
  }

  // [lo, hi] around the k-th largest fp32 score: linear bins over the range, then over the bin
  // that holds it, until it is known or the range cannot be cut any more
  int need = k;
  while (lo < hi) {
    const float base = 0.5f * lo, inv = (float)(SEL_BINS - 1) / (0.5f * hi - base);
    if (!(inv < SEL_MAX)) break;
    auto bin_of = [&](float x) { return min((int)((0.5f * x - base) * inv), SEL_BINS - 1); };
    __syncthreads();
    for (int i = tid; i < SEL_BINS; i += THREADS) sh.bins[i] = 0;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    for (int j = tid; j < n; j += THREADS) {
      const float x = x_of[j];
      if (x >= lo && x <= hi) atomicAdd(&sh.bins[bin_of(x)], 1u);
    }
    __syncthreads();
    // counts from the top: thread i owns bins [top - (i + 1) PER, top - i PER)
    constexpr int PER = SEL_BINS / THREADS;
    uint32_t c[PER];
    int sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      c[i] = sh.bins[SEL_BINS - 1 - (tid * PER + i)];
      sum += (int)c[i];
    }
    int incl = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(incl, off, 64);
      if (lane >= off) incl += v;
    }
    if (lane == 63) sh.wave_a[wave] = incl;
    __syncthreads();
    int before = incl - sum;
    for (int w = 0; w < wave; ++w) before += sh.wave_a[w];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (before < need && need <= before + (int)c[i]) {
        sh.found = SEL_BINS - 1 - (tid * PER + i);
        sh.below = before;
        sh.in_bin = (int)c[i];
      }
      before += (int)c[i];
    }
    __syncthreads();
    const int bin = sh.found, in_bin = sh.in_bin;
    need -= sh.below;
    if (in_bin <= SEL_LIST) {
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
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      l2 = fminf(l2, __shfl_xor(l2, off, 64));
      h2 = fmaxf(h2, __shfl_xor(h2, off, 64));
    }
    if (lane == 0) {
      sh.wave_lo[wave] = l2;
      sh.wave_hi[wave] = h2;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      l2 = fminf(l2, sh.wave_lo[w]);
      h2 = fmaxf(h2, sh.wave_hi[w]);
    }
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
      if (i < SEL_LIST) sh.list_j[i] = j;
    }
  }
  sure = block_sum<THREADS>(sure, sh.wave_a);
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
  if (close <= SEL_LIST) {
    for (int i = wave; i < close; i += WAVES) {
      const double s = score64<T, FP8>(a, p, t, table, sh.list_j[i], lane);
      if (lane == 0) sh.list_key[i] = order_of(s);
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
  // largest 64-bit score by its bytes, the scores formed again for each
  uint64_t prefix = 0;
  int want = rest;
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += THREADS) sh.bins[i] = 0;
    __syncthreads();
    for (int j = wave; j < n; j += WAVES) {
      const float x = x_of[j];
      if (!(x >= b_lo && x <= b_hi) || x == SEL_NONE) continue;
      const uint64_t key = order_of(score64<T, FP8>(a, p, t, table, j, lane));
      if (lane == 0 && (shift == 56 || key >> (shift + 8) == prefix))
        atomicAdd(&sh.bins[(key >> shift) & 255], 1u);
    }
    __syncthreads();
    int digit = 255, above = 0;
    while (digit > 0 && above + (int)sh.bins[digit] < want) above += (int)sh.bins[digit--];
    want -= above;
    prefix = (prefix << 8) | (uint64_t)digit;
    __syncthreads();
  }
  for (int j = wave; j < n; j += WAVES) {
    const float x = x_of[j];
    float y = x > b_hi ? taken_x : SEL_NONE;
    if (x >= b_lo && x <= b_hi && x != SEL_NONE) {
      const uint64_t key = order_of(score64<T, FP8>(a, p, t, table, j, lane));
      y = key > prefix ? taken_x : key == prefix ? SEL_MAX : SEL_NONE;
    }
    if (lane == 0) x_of[j] = y;
  }
  __syncthreads();
  emit([&](int j) { return x_of[j] > SEL_MAX; }, [&](int j) { return x_of[j] == SEL_MAX; }, want);
}

// ---------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------

// Scores of a pass may take this much of the workspace; more query rows take more passes.
constexpr int64_t SEL_PASS_BYTES = 512ll << 20;

struct PassPlan {
  SelPlan p;
  bool tiles;          // score_tile_kernel
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
  r.tiles = per_seq >= 4;
  p.wq = r.tiles ? TILE_WAVES : per_seq >= 2 ? 2 : 1;
  p.slices = r.tiles ? 1 : 4 / p.wq;
  const int64_t groups = (r.rows + p.wq - 1) / p.wq;
  if (r.tiles) {
    p.chunk = 512;
  } else {
    int64_t c = (int64_t)p.width * groups / 2048;
    const int unit = 64 * p.slices;
    c = (c + unit - 1) / unit * unit;
    p.chunk = (int)(c < unit ? unit : c > 2048 ? 2048 : c);
  }
  p.chunks = (p.width + p.chunk - 1) / p.chunk;
  // every part starts on 16 bytes
  const int64_t w_floats = ((int64_t)r.rows + 3) / 4 * 4;
  const int64_t k_floats = ((int64_t)a.batch * p.chunks * p.slices + 3) / 4 * 4;
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
  if (a->key_format == SAS_ROW_FP8_INDEX && (int64_t)a->block_size * (a->dim + 4) % 16) {
    return fail("fp8 index pages must be a multiple of 16 bytes");
  }
  if (a->rows_per_seq > 0 && (int64_t)a->rows_per_seq * a->batch != a->tokens) {
    return fail("tokens must be batch * rows_per_seq");
  }
  return SAS_OK;
}

template <typename T, bool FP8, int D, int MT>
void launch_scores(const SasSelectArgs& a, const PassPlan& r, const SelPlan& p, hipStream_t st) {
  const int64_t groups = (p.t_end - p.t_begin + p.wq - 1) / p.wq;
  const dim3 grid((unsigned)(groups * p.chunks));
  if (r.tiles) {
    hipLaunchKernelGGL((score_tile_kernel<T, FP8, D, MT>), grid, dim3(64 * TILE_WAVES), 0, st, a, p);
  } else {
    hipLaunchKernelGGL((score_stream_kernel<T, FP8, D, MT>), grid, dim3(256), 0, st, a, p);
  }
}

template <typename T, bool FP8>
void launch_pass(const SasSelectArgs& a, const PassPlan& r, const SelPlan& p, hipStream_t st) {
  if (a.max_keys > a.topk) {  // else every row takes all it may see: no scores
    const int mt = (a.heads + 31) / 32;
    if (a.dim == 128) {
      if (mt == 1) launch_scores<T, FP8, 128, 1>(a, r, p, st);
      else if (mt == 2) launch_scores<T, FP8, 128, 2>(a, r, p, st);
      else launch_scores<T, FP8, 128, 4>(a, r, p, st);
    } else {
      if (mt == 1) launch_scores<T, FP8, 64, 1>(a, r, p, st);
      else if (mt == 2) launch_scores<T, FP8, 64, 2>(a, r, p, st);
      else launch_scores<T, FP8, 64, 4>(a, r, p, st);
    }
  }
  const dim3 grid((unsigned)(p.t_end - p.t_begin));
  if (a.max_keys <= 4096) {
    hipLaunchKernelGGL((select_kernel<T, FP8, 256, 4096>), grid, dim3(256), 0, st, a, p);
  } else if (a.max_keys <= 32768) {
    hipLaunchKernelGGL((select_kernel<T, FP8, 1024, 32768>), grid, dim3(1024), 0, st, a, p);
  } else {
    hipLaunchKernelGGL((select_kernel<T, FP8, 1024, 0>), grid, dim3(1024), 0, st, a, p);
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
      fp8 ? sas::launch_pass<__bf16, true>(*a, r, p, st) : sas::launch_pass<__bf16, false>(*a, r, p, st);
    } else {
      fp8 ? sas::launch_pass<_Float16, true>(*a, r, p, st)
          : sas::launch_pass<_Float16, false>(*a, r, p, st);
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
