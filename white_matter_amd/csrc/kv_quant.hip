// Quantised KV pool for gfx950: the store (key norm, weight, RoPE, quantising
// and the slot scatter in one pass over keys and values) and the read-back
// (formats and formulas in wmx_attn.h). HBM-bound: each thread moves 8
// consecutive elements of a row, 16 or 32 bytes in and 8 out. Measured, 8 x 8
// channels x 16 heads x 2,048 tokens of 64 from bf16 to e4m3: 829 MB in 167 us
// (5.0 TB/s, a large copy's 4.8); one token of 8 rows of 8 x 8 heads 4.6 us. The
// read-back of 4 x 8 x 8 x 4,096 rows of 128: 407 MB in 84 us (4.8 TB/s).
#include "wmx_kernels.h"

namespace wmx {

constexpr float kSmallestRow = 0x1p-100f;  // rows whose magnitudes stay below are stored as zeros

template <int FMT>
__device__ __forceinline__ constexpr float largest_code() { return FMT == WMX_POOL_E4M3 ? 448.f : 127.f; }

// Eight scaled values (magnitudes up to the largest code and a rounding) as
// codes, to nearest even. Neither conversion can pass its range: a magnitude
// within a rounding of the largest code rounds to it.
template <int FMT>
__device__ __forceinline__ u32x2 to_codes(const float (&y)[8]) {
  u32x2 r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (FMT == WMX_POOL_E4M3) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], w, true);
      r[h] = (uint32_t)w;
    } else {
      uint32_t w = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) w |= ((uint32_t)(int)__builtin_rintf(y[4 * h + e]) & 0xffu) << (8 * e);
      r[h] = w;
    }
  }
  return r;
}

// The codes of a row held by L lanes, 8 values each, and its scale. The
// magnitudes are compared as integers, where infinities and NaN are largest.
template <int FMT, int L>
__device__ __forceinline__ u32x2 quantise_row(float (&x)[8], float& scale) {
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = __float_as_uint(x[e]) & 0x7fffffffu;
    most = most > b ? most : b;
  }
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    const uint32_t b = __shfl_xor(most, o);
    most = most > b ? most : b;
  }
  constexpr float kTop = largest_code<FMT>();
  const float a = __uint_as_float(most);
  const bool finite = most < 0x7f800000u;
  const bool live = finite && a >= kSmallestRow;
  const float inv = live ? kTop / a : 0.f;
  scale = live ? a / kTop : finite ? 0.f : __builtin_nanf("");
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = live ? x[e] * inv : 0.f;
  return to_codes<FMT>(x);
}

// One (b, c, t, head group) per L consecutive lanes (token-fastest, so
// neighbouring lanes read and write neighbouring rows); each thread walks its
// group's heads, one at a time: 71 registers leave seven waves a SIMD, whose loads
// overlap (the 829 MB above with four heads' loads in flight 197 us, and few heads
// per thread 20 us where one at a time takes 9.6).
template <int D, int FMT, bool KEY, bool VALUE>
__global__ __launch_bounds__(256) void kv_quant_kernel(const wmx_kv_quant_args a, int64_t tokens_total, int head_groups) {
  constexpr int LD = D / 8;           // lanes holding data
  constexpr int L = LD <= 8 ? 8 : 16; // lanes per row (a power of two; D = 96 leaves 4 idle)
  const int64_t gid = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t unit = gid / L;
  const int l = (int)(gid % L);
  const int64_t r = unit / head_groups;
  const int hg = (int)(unit - r * head_groups);
  // a row's L lanes share r and hg: they leave together, before any exchange
  if (r >= tokens_total) return;
  const int t = (int)(r % a.tokens);
  const int64_t bc = r / a.tokens;
  const int c = (int)(bc % a.channels);
  const int b = (int)(bc / a.channels);
  const int per_group = (a.heads + head_groups - 1) / head_groups;
  const int h_begin = hg * per_group, h_end = min(h_begin + per_group, a.heads);
  if (h_begin >= h_end) return;
  const int64_t slot = a.slots ? a.slots[(int64_t)b * a.slots_stride + t] : t;
  const bool slot_ok = slot >= 0 && slot < a.pool_slots;
  const int d0 = 8 * l;
  const bool data = l < LD;
  const int dl = data ? d0 : 0;

  float w[8], cs[8], sn[8];
  if constexpr (KEY) {
    load8(a.k_norm_weight, (int64_t)c * D + dl, a.weight_dtype == WMX_DTYPE_BF16, w);
    const int64_t ro = a.rope_by_slot ? (slot_ok ? slot : 0) * a.rope_stride[1] + dl
                                      : (int64_t)b * a.rope_stride[0] + (int64_t)t * a.rope_stride[1] + dl;
    load8(a.cos, ro, a.rope_dtype == WMX_DTYPE_BF16, cs);
    load8(a.sin, ro, a.rope_dtype == WMX_DTYPE_BF16, sn);
  }
  // rotate_half: element d pairs with d +- D/2, held by the lane LD/2 away
  const bool low = d0 < D / 2;
  const int partner = (int)(gid & 63) + (low ? LD / 2 : -(LD / 2));
  const auto row_of = [&](const int64_t* st, int64_t n) { return (int64_t)b * st[0] + (int64_t)c * st[1] + n * st[3]; };
  const int64_t key_row = row_of(a.key_stride, t) + dl, value_row = row_of(a.value_stride, t) + dl;

  for (int h = h_begin; h < h_end; ++h) {
    float x[8], v[8];
    if constexpr (KEY) load8<true>(a.key, key_row + h * a.key_stride[2], a.key_dtype == WMX_DTYPE_BF16, x);
    if constexpr (VALUE) load8<true>(a.value, value_row + h * a.value_stride[2], a.value_dtype == WMX_DTYPE_BF16, v);
    __builtin_amdgcn_sched_barrier(0);  // keep both loads ahead of the first use
    const auto put = [&](float (&row)[8], void* codes, const int64_t* cst, float* scales, const int64_t* sst) {
      if (!data) {
#pragma unroll
        for (int e = 0; e < 8; ++e) row[e] = 0.f;  // idle lanes (D = 96)
      }
      float scale;
      const u32x2 code = quantise_row<FMT, L>(row, scale);
      if (data && slot_ok) {
        const int64_t at = row_of(cst, slot) + h * cst[2] + d0;
        __builtin_nontemporal_store(code, (u32x2*)((char*)codes + at));
        if (l == 0) scales[row_of(sst, slot) + h * sst[2]] = scale;
      }
    };
    if constexpr (KEY) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
      if (!data) ss = 0.f;
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
      const float inv = 1.f / sqrtf(ss / (float)D + a.eps);
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = x[e] * inv * w[e];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float other = __shfl(y[e], data ? partner : 0);
        x[e] = fmaf(low ? -other : other, sn[e], y[e] * cs[e]);
      }
      put(x, a.key_codes, a.key_codes_stride, a.key_scales, a.key_scales_stride);
    }
    if constexpr (VALUE) put(v, a.value_codes, a.value_codes_stride, a.value_scales, a.value_scales_stride);
  }
}

template <int D, int FMT>
static void launch_kv_quant_d(const wmx_kv_quant_args& a, int64_t rows, int groups, dim3 grid, hipStream_t stream) {
  if (!a.key)
    hipLaunchKernelGGL((kv_quant_kernel<D, FMT, false, true>), grid, dim3(256), 0, stream, a, rows, groups);
  else if (a.value)
    hipLaunchKernelGGL((kv_quant_kernel<D, FMT, true, true>), grid, dim3(256), 0, stream, a, rows, groups);
  else
    hipLaunchKernelGGL((kv_quant_kernel<D, FMT, true, false>), grid, dim3(256), 0, stream, a, rows, groups);
}

int launch_kv_quant(const wmx_kv_quant_args& a, hipStream_t stream) {
  const int64_t rows = (int64_t)a.batch * a.channels * a.tokens;
  if (rows == 0 || a.heads == 0) return WMX_OK;
  const int64_t lanes = a.head_dim <= 64 ? 8 : 16;
  // threads walk all heads of a token where that still gives every CU four
  // workgroups; fewer rows (a decode step) split the heads (the 829 MB with a head
  // a thread 258 us; 251 tokens of 3 x 4 channels x 6 heads of 96 9.4 us, 10.6 with
  // a workgroup a CU)
  int64_t groups = 1;
  while (groups < a.heads && rows * groups * lanes < 1024 * 256) groups *= 2;
  if (groups > a.heads) groups = a.heads;
  const int64_t blocks = (rows * groups * lanes + 255) / 256;
  if (blocks > INT32_MAX) return WMX_E_UNSUPPORTED;
  const dim3 grid((unsigned)blocks);
  const bool e4m3 = a.format == WMX_POOL_E4M3;
  switch (a.head_dim) {
    case 64:
      if (e4m3) launch_kv_quant_d<64, WMX_POOL_E4M3>(a, rows, (int)groups, grid, stream);
      else launch_kv_quant_d<64, WMX_POOL_INT8>(a, rows, (int)groups, grid, stream);
      return WMX_OK;
    case 96:
      if (e4m3) launch_kv_quant_d<96, WMX_POOL_E4M3>(a, rows, (int)groups, grid, stream);
      else launch_kv_quant_d<96, WMX_POOL_INT8>(a, rows, (int)groups, grid, stream);
      return WMX_OK;
    case 128:
      if (e4m3) launch_kv_quant_d<128, WMX_POOL_E4M3>(a, rows, (int)groups, grid, stream);
      else launch_kv_quant_d<128, WMX_POOL_INT8>(a, rows, (int)groups, grid, stream);
      return WMX_OK;
    default: return WMX_E_UNSUPPORTED;
  }
}

// ----------------------------------------------------------- read-back ----
// Eight codes per thread: consecutive threads take consecutive parts of a row,
// then consecutive tokens.
template <int FMT>
__global__ __launch_bounds__(256) void kv_read_kernel(const wmx_kv_read_args a, int64_t vectors) {
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (gid >= vectors) return;
  const int per_row = a.head_dim / 8;
  const int64_t row = gid / per_row;
  const int d0 = 8 * (int)(gid - row * per_row);
  int64_t rest = row / a.tokens;
  const int64_t t = row - rest * a.tokens;
  const int64_t h = rest % a.heads;
  rest /= a.heads;
  const int64_t c = rest % a.channels, b = rest / a.channels;
  const int64_t slot = a.slots ? a.slots[b * a.slots_stride + t] : t;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.f;
  if (slot >= 0 && slot < a.pool_slots) {
    const int64_t at = b * a.codes_stride[0] + c * a.codes_stride[1] + h * a.codes_stride[2] + slot * a.codes_stride[3] + d0;
    const u32x2 w = __builtin_nontemporal_load((const u32x2*)((const char*)a.codes + at));
    const float scale =
        a.scales[b * a.scales_stride[0] + c * a.scales_stride[1] + h * a.scales_stride[2] + slot * a.scales_stride[3]];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (FMT == WMX_POOL_E4M3) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
        x[4 * i] = lo[0] * scale;
        x[4 * i + 1] = lo[1] * scale;
        x[4 * i + 2] = hi[0] * scale;
        x[4 * i + 3] = hi[1] * scale;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * i + e] = (float)(int8_t)(w[i] >> (8 * e)) * scale;
      }
    }
  }
  store8_bf16(a.out, row * a.head_dim + d0, x);
}

int launch_kv_read(const wmx_kv_read_args& a, hipStream_t stream) {
  const int64_t vectors = (int64_t)a.batch * a.channels * a.heads * a.tokens * (a.head_dim / 8);
  if (vectors == 0) return WMX_OK;
  const int64_t blocks = (vectors + 255) / 256;
  if (blocks > INT32_MAX) return WMX_E_UNSUPPORTED;
  if (a.format == WMX_POOL_E4M3)
    hipLaunchKernelGGL((kv_read_kernel<WMX_POOL_E4M3>), dim3((unsigned)blocks), dim3(256), 0, stream, a, vectors);
  else
    hipLaunchKernelGGL((kv_read_kernel<WMX_POOL_INT8>), dim3((unsigned)blocks), dim3(256), 0, stream, a, vectors);
  return WMX_OK;
}

}  // namespace wmx
