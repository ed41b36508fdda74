// Row operators around the attention call: the norm and the rotation of query heads, and the
// same for new cache rows on their way into a paged cache (no reference counterpart: the
// reference takes rotated queries and written caches, api.py:129-153).
//
// A row x of D dims becomes
//   y[d] = x[d] * rsqrt(mean(x[0..N)^2) + eps) * w[d]   for d < N (N = 0: no norm), x[d] behind it
// and then the pairs of dims [off, off + R) are turned by the angle of the row's position:
//   (a, b) -> (a cos - b sin, b cos + a sin)
// with pair i = dims (2i, 2i + 1) of the range (interleaved) or (i, i + R / 2) (halves), and
// cos / sin from the caller's fp32 table. Everything is in fp32 and rounded once, at the store; rows
// that end in fp8 are in 64 bits up to their codes, whose coarse steps would otherwise turn an
// fp32 rounding into a whole step now and then (128 rows of 656 bytes: 4.7 us, in fp32 4.6).
//
// Bound by memory: a row is read once and written once. A group of G lanes (8 to 64, the fewest
// that hold the row at 16 bytes a lane, two or four loads a lane above 512 dims) owns a row, so
// the sum of squares is a reduction inside the group and a wave of short rows works on several.
// All of a row's loads come before its stores and no other lane touches the row, so the result
// may go to where the row came from.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/sas_mi355x.h"

namespace sas {

void set_error(const std::string& msg);

namespace {

constexpr float ROWS_E4M3_MAX = 448.0f;
constexpr int ROWS_WG = 256;

enum RowOut { OUT_HEADS = 0, OUT_CACHE = 1, OUT_FP8_MLA = 2, OUT_FP8_INDEX = 3 };

template <typename T>
struct Vec8 {
  typedef T type __attribute__((ext_vector_type(8)));
};

template <typename T, typename W>
__device__ inline void load8(const void* p, W f[8]) {
  const typename Vec8<T>::type v = *(const typename Vec8<T>::type*)p;
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (W)(float)v[i];
}

template <typename W>
__device__ inline void load8f(const float* p, W f[8]) {
  const float4 a = ((const float4*)p)[0], b = ((const float4*)p)[1];
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
  f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

template <typename T, typename W>
__device__ inline void norm_weight8(const SasRowArgs& a, int e0, W w[8]) {
  if (a.norm_weight_fp32) {
    load8f((const float*)a.norm_weight + e0, w);
  } else {
    load8<T>((const T*)a.norm_weight + e0, w);
  }
}

template <int OUT>
struct WideOf {
  typedef float type;
};
template <>
struct WideOf<OUT_FP8_MLA> {
  typedef double type;
};
template <>
struct WideOf<OUT_FP8_INDEX> {
  typedef double type;
};

template <typename T, int G, int NCH, int OUT>
__global__ __launch_bounds__(ROWS_WG) void rows_kernel(SasRowArgs a) {
  const int lane = threadIdx.x & (G - 1);
  const int64_t row = (int64_t)blockIdx.x * (ROWS_WG / G) + threadIdx.x / G;
  if (row >= (int64_t)a.tokens * a.heads) return;
  // (fewer than 2^31 rows: a 32-bit division)
  const int t = OUT == OUT_HEADS ? (int)((uint32_t)row / (uint32_t)a.heads) : (int)row;
  const int h = OUT == OUT_HEADS ? (int)row - t * a.heads : 0;
  int64_t slot = 0;
  if (OUT != OUT_HEADS) {
    slot = a.slots[t];
    if (slot < 0 || slot >= a.cache_rows) return;
  }
  const T* x = (const T*)a.x + (int64_t)t * a.x_token_stride + (int64_t)h * a.x_head_stride;
  const int chunks = a.dim >> 3;

  typedef typename WideOf<OUT>::type W;
  W f[NCH][8];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = lane + i * G;
    if (c < chunks) {
      load8<T>(x + 8 * c, f[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[i][e] = 0;
    }
  }
  // the other members of the halves' pairs, before anything is stored
  const int r0 = a.rope_offset, r1 = r0 + a.rope_dim, half = a.rope_dim >> 1;
  W p[NCH][8];
  if (!a.interleaved) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int e0 = 8 * (lane + i * G);
      if (e0 >= r0 && e0 < r1) load8<T>(x + (e0 - r0 < half ? e0 + half : e0 - half), p[i]);
    }
  }

  if (a.norm_dim > 0) {
    W s = 0;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (8 * (lane + i * G) < a.norm_dim) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fma(f[i][e], f[i][e], s);
      }
    }
#pragma unroll
    for (int off = 1; off < G; off <<= 1) s += __shfl_xor(s, off, 64);
    const W inv = (W)1 / sqrt(s / (W)a.norm_dim + (W)a.eps);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int e0 = 8 * (lane + i * G);
      W w[8];
      if (e0 < a.norm_dim) {
        norm_weight8<T>(a, e0, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[i][e] = f[i][e] * inv * w[e];
      }
      if (!a.interleaved && e0 >= r0 && e0 < r1) {
        const int q0 = e0 - r0 < half ? e0 + half : e0 - half;
        if (q0 < a.norm_dim) {
          norm_weight8<T>(a, q0, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) p[i][e] = p[i][e] * inv * w[e];
        }
      }
    }
  }

  if (a.rope_dim > 0) {
    const int pos = a.positions[t];
    const bool in_table = pos >= 0 && pos < a.max_position;
    const float* cs = a.cos_sin + (int64_t)(in_table ? pos : 0) * a.rope_dim;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int e0 = 8 * (lane + i * G);
      if (e0 < r0 || e0 >= r1) continue;
      W c[8], s[8];
      if (a.interleaved) {
        const float4 cv = *(const float4*)(cs + ((e0 - r0) >> 1));
        const float4 sv = *(const float4*)(cs + half + ((e0 - r0) >> 1));
        c[0] = cv.x, c[1] = cv.y, c[2] = cv.z, c[3] = cv.w;
        s[0] = sv.x, s[1] = sv.y, s[2] = sv.z, s[3] = sv.w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const W u = f[i][2 * j], v = f[i][2 * j + 1];
          f[i][2 * j] = u * c[j] - v * s[j];
          f[i][2 * j + 1] = v * c[j] + u * s[j];
        }
      } else {
        const bool first = e0 - r0 < half;
        const int k0 = first ? e0 - r0 : e0 - r0 - half;
        load8f(cs + k0, c);
        load8f(cs + half + k0, s);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          f[i][e] = first ? f[i][e] * c[e] - p[i][e] * s[e] : f[i][e] * c[e] + p[i][e] * s[e];
      }
      if (!in_table) {
        // a position without angles has no rotation: not a number, rather than another's
#pragma unroll
        for (int e = 0; e < 8; ++e) f[i][e] = (W)__builtin_nanf("");
      }
    }
  }

  if (OUT == OUT_HEADS || OUT == OUT_CACHE) {
    T* o = OUT == OUT_HEADS
               ? (T*)a.out + (int64_t)t * a.out_token_stride + (int64_t)h * a.out_head_stride
               : (T*)a.out + slot * a.dim;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = lane + i * G;
      if (c < chunks) {
        typename Vec8<T>::type v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (T)f[i][e];
        *(typename Vec8<T>::type*)(o + 8 * c) = v;
      }
    }
    return;
  }

  // fp8 rows: one scale per 128 dims (16 lanes) of the 512 latent dims, or one per index row
  constexpr int SCALE_LANES = OUT == OUT_FP8_MLA ? 16 : G;
  // Dims that nothing has changed are quantized as sas_kv_fp8_append does (fp32 scale and quotient);
  // others from their 64-bit values, so that only the code's own rounding is left.
  const bool raw = a.norm_dim == 0 && (a.rope_dim == 0 || (OUT == OUT_FP8_MLA && a.rope_offset >= 512));
  bool bad = false;  // (the maximum drops NaN: a row with one gets a NaN scale)
  float y[8], stored;
#pragma unroll
  for (int e = 0; e < 8; ++e) bad |= f[0][e] != f[0][e];
  if (raw) {
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf((float)f[0][e]));
    if (bad) amax = __builtin_inff();
#pragma unroll
    for (int off = 1; off < SCALE_LANES; off <<= 1) amax = fmaxf(amax, __shfl_xor(amax, off, 64));
    stored = amax > 0.0f ? amax / ROWS_E4M3_MAX : 1.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (float)f[0][e] / stored;
  } else {
    double amax = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmax(amax, fabs((double)f[0][e]));
    if (bad) amax = (double)__builtin_inff();
#pragma unroll
    for (int off = 1; off < SCALE_LANES; off <<= 1) amax = fmax(amax, __shfl_xor(amax, off, 64));
    stored = amax > 0.0 ? (float)(amax / (double)ROWS_E4M3_MAX) : 1.0f;
    const double inv = amax > 0.0 ? (double)ROWS_E4M3_MAX / amax : 1.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (float)((double)f[0][e] * inv);
  }
  if (!(stored < __builtin_inff())) stored = __builtin_nanf("");
  uint32_t packed[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = fminf(fmaxf(y[4 * k + e], -ROWS_E4M3_MAX), ROWS_E4M3_MAX);
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
    packed[k] = (uint32_t)w;
  }
  if (OUT == OUT_FP8_MLA) {
    unsigned char* o = (unsigned char*)a.out + slot * SAS_FP8_ROW_BYTES;
    *(uint2*)(o + 8 * lane) = make_uint2(packed[0], packed[1]);
    if ((lane & 15) == 0) *(float*)(o + 512 + 4 * (lane >> 4)) = stored;
    if (lane < 8) {
      typename Vec8<T>::type v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (T)(float)f[NCH - 1][e];
      *(typename Vec8<T>::type*)(o + 528 + 16 * lane) = v;
    }
  } else if (lane < chunks) {
    // a page of block_size rows: their codes, then their scales
    const int64_t page = slot / a.block_size, at = slot - page * a.block_size;
    unsigned char* o = (unsigned char*)a.out + page * a.block_size * (a.dim + 4);
    *(uint2*)(o + at * a.dim + 8 * lane) = make_uint2(packed[0], packed[1]);
    if (lane == 0) *(float*)(o + a.block_size * (int64_t)a.dim + 4 * at) = stored;
  }
}

template <typename T, int G, int NCH, int OUT>
int launch_rows(const SasRowArgs& a, void* stream, const char* who) {
  const int64_t rows = (int64_t)a.tokens * a.heads;
  const int64_t grid = (rows + ROWS_WG / G - 1) / (ROWS_WG / G);
  hipLaunchKernelGGL((rows_kernel<T, G, NCH, OUT>), dim3((unsigned)grid), dim3(ROWS_WG), 0,
                     (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error(std::string(who) + ": " + hipGetErrorString(e));
    return SAS_E_HIP;
  }
  return SAS_OK;
}

template <typename T, int OUT>
int launch_by_width(const SasRowArgs& a, void* stream, const char* who) {
  const int chunks = a.dim >> 3;
  if (chunks <= 8) return launch_rows<T, 8, 1, OUT>(a, stream, who);
  if (chunks <= 16) return launch_rows<T, 16, 1, OUT>(a, stream, who);
  if (chunks <= 32) return launch_rows<T, 32, 1, OUT>(a, stream, who);
  if (chunks <= 64) return launch_rows<T, 64, 1, OUT>(a, stream, who);
  return launch_rows<T, 64, 2, OUT>(a, stream, who);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_rows(const SasRowArgs* a, const char* who) {
  auto fail = [&](const char* what) {
    set_error(std::string(who) + ": " + what);
    return SAS_E_INVALID;
  };
  if (!a) return fail("null arguments");
  if (a->tokens < 0 || a->heads < 1) return fail("negative size");
  if ((int64_t)a->tokens * a->heads >= (1ll << 31)) return fail("2^31 rows or more");
  if (a->dim < 8 || a->dim > SAS_ROW_MAX_DIM || a->dim % 8) return fail("dim must be a multiple of 8 up to 1024");
  if (a->dtype != SAS_DTYPE_BF16 && a->dtype != SAS_DTYPE_FP16) return fail("dtype");
  if (a->norm_dim < 0 || a->norm_dim > a->dim || a->norm_dim % 8) return fail("norm_dim must be a multiple of 8 up to dim");
  if (a->rope_dim < 0 || a->rope_offset < 0 || a->rope_dim % (a->interleaved ? 8 : 16) ||
      a->rope_offset % 8 || a->rope_dim > a->dim || a->rope_offset > a->dim - a->rope_dim) {
    return fail("rotated dims out of the row, or not in whole groups");
  }
  if (a->tokens == 0) return SAS_OK;
  if (!a->x || !a->out || (a->norm_dim && !a->norm_weight) ||
      (a->rope_dim && (!a->positions || !a->cos_sin))) {
    return fail("null pointer");
  }
  if (a->rope_dim && a->max_position < 1) return fail("empty angle table");
  if (!aligned16(a->x) || !aligned16(a->out) || !aligned16(a->cos_sin) || !aligned16(a->norm_weight) ||
      a->x_token_stride % 8 || a->x_head_stride % 8) {
    return fail("rows must be aligned to 16 bytes");
  }
  return SAS_OK;
}

}  // namespace
}  // namespace sas

extern "C" int sas_norm_rope(const SasRowArgs* a, void* stream) {
  const char* who = "sas_norm_rope";
  const int rc = sas::check_rows(a, who);
  if (rc != SAS_OK || a->tokens == 0) return rc;
  if (a->out_token_stride % 8 || a->out_head_stride % 8) {
    sas::set_error("sas_norm_rope: rows must be aligned to 16 bytes");
    return SAS_E_INVALID;
  }
  return a->dtype == SAS_DTYPE_BF16 ? sas::launch_by_width<__bf16, sas::OUT_HEADS>(*a, stream, who)
                                    : sas::launch_by_width<_Float16, sas::OUT_HEADS>(*a, stream, who);
}

extern "C" int sas_kv_append_rope(const SasRowArgs* a, void* stream) {
  const char* who = "sas_kv_append_rope";
  const int rc = sas::check_rows(a, who);
  if (rc != SAS_OK) return rc;
  auto fail = [&](const char* what) {
    sas::set_error(std::string(who) + ": " + what);
    return (int)SAS_E_INVALID;
  };
  if (a->heads != 1) return fail("cache rows have one head");
  if (a->cache_rows < 0) return fail("negative size");
  if (a->row_format == SAS_ROW_FP8_DS_MLA) {
    if (a->dim != 576 || a->dtype != SAS_DTYPE_BF16) return fail("656-byte rows hold 576 bf16 dims");
  } else if (a->row_format == SAS_ROW_FP8_INDEX) {
    if (a->dim != 64 && a->dim != 128) return fail("fp8 index rows hold 64 or 128 dims");
    if (a->block_size < 1 || a->cache_rows % a->block_size) return fail("whole pages of block_size rows");
    // (a page is block_size * (dim + 4) bytes: its codes and scales are aligned when this is)
    if ((int64_t)a->block_size * (a->dim + 4) % 16) return fail("fp8 index pages must be a multiple of 16 bytes");
  } else if (a->row_format != SAS_ROW_NATIVE) {
    return fail("row_format");
  }
  if (a->tokens == 0) return SAS_OK;
  if (!a->slots) return fail("null pointer");
  if (a->row_format == SAS_ROW_FP8_DS_MLA) {
    return sas::launch_rows<__bf16, 64, 2, sas::OUT_FP8_MLA>(*a, stream, who);
  }
  if (a->row_format == SAS_ROW_FP8_INDEX) {
    if (a->dtype == SAS_DTYPE_BF16) {
      return a->dim == 64 ? sas::launch_rows<__bf16, 8, 1, sas::OUT_FP8_INDEX>(*a, stream, who)
                          : sas::launch_rows<__bf16, 16, 1, sas::OUT_FP8_INDEX>(*a, stream, who);
    }
    return a->dim == 64 ? sas::launch_rows<_Float16, 8, 1, sas::OUT_FP8_INDEX>(*a, stream, who)
                        : sas::launch_rows<_Float16, 16, 1, sas::OUT_FP8_INDEX>(*a, stream, who);
  }
  return a->dtype == SAS_DTYPE_BF16 ? sas::launch_by_width<__bf16, sas::OUT_CACHE>(*a, stream, who)
                                    : sas::launch_by_width<_Float16, sas::OUT_CACHE>(*a, stream, who);
}

extern "C" int sas_row_args_struct_size(void) { return (int)sizeof(SasRowArgs); }
