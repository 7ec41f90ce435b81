// Attention of drafted tokens (a tree, or one token) over a bf16 or quantised
// KV pool for gfx950 (visibility and formats in wmx_attn.h).
//
// The query rows of one KV head (nodes x query heads of its group, node-major)
// share its keys and values, so a workgroup takes 16 MB of them and a range of
// slots; each K/V byte is read from HBM once per row tile and converted once.
// Four waves take every fourth 32-slot tile of the range and keep their own
// running maximum, sum and output, merged through LDS at the end; ranges of
// one row are merged by a second kernel in log-sum-exp form.
//
// Nothing is staged in LDS: with v_mfma_f32_16x16x32_bf16
//   S^T = K Q^T    A: lane l holds key l % 16, 8 consecutive d of its quarter
//                  l / 16; the d order is the one in which its loads are
//                  widest, the same for Q
//   O^T = V^T P^T  B: P as S^T left it in the accumulators: lane (query l % 16,
//                  quarter q) holds keys 4 q + [0, 4) of the tile's two
//                  16-key halves; A: V of those keys, loaded as D/16
//                  consecutive d per lane and transposed between registers
//                  (v_perm), so output block c holds d = (D/16) i + c
// K and V scales multiply scores and weights, one operation per score instead
// of one per element; codes are converted exactly to bf16.
#include <climits>

#include "wmx_kernels.h"

namespace wmx {

constexpr int kTreeWaves = 4;
constexpr int kTreeTile = 32;                          // slots per wave and step
constexpr int kTreeStep = kTreeWaves * kTreeTile;      // slots per workgroup and step

__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}

// Two codes (the low or high half of a dword) as a bf16 pair, exactly.
template <int FMT, bool HIGH>
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  if constexpr (FMT == WMX_POOL_E4M3) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
  } else {
    const int s = HIGH ? 16 : 0;
    return pack_bf16x2((float)(int8_t)(w >> s), (float)(int8_t)(w >> (s + 8)));
  }
}

// How a wave reads 32 slots of K and V.
template <int FMT, int D>
struct TreeTile {
  static constexpr int kElem = FMT == WMX_POOL_BF16 ? 2 : 1;  // bytes
  static constexpr int KS = D / 32;                           // k-steps of S^T
  static constexpr int W = D / 16;                            // consecutive d per lane of V
  // A lane's K operand of k-step s: bf16 and D = 96 codes take 8 d at
  // 8 (q + 4 s); other codes 16 bytes, two k-steps, at 16 (q + 4 (s / 2)).
  static constexpr bool kWide = FMT != WMX_POOL_BF16 && D % 64 == 0;
  static constexpr int KD = FMT == WMX_POOL_BF16 ? 4 : 2;     // dwords of 8 d
  static constexpr int VD = W * kElem / 4 + (W * kElem % 4 ? 1 : 0);  // dwords of W d

  static __device__ __forceinline__ int k_dim(int s, int q) {
    return kWide ? 16 * (q + 4 * (s / 2)) + 8 * (s % 2) : 8 * (q + 4 * s);
  }
  // first d of output block c, row index i of the block
  static __device__ __forceinline__ int v_dim(int i, int c) {
    if constexpr (FMT != WMX_POOL_BF16 && D == 96) return c < 4 ? 4 * i + c : 64 + 2 * i + (c - 4);
    else return W * i + c;
  }

  uint32_t k[2][KS][KD];  // key halves
  uint32_t v[8][VD];      // the lane's keys: 4 q + (e & 3) + 16 (e >> 2)

  // lk(row), lv(row): byte offset of a tile row from the (wave-uniform) base
  template <class Row>
  __device__ __forceinline__ void load_k(const char* base, int li, int q, Row row) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const char* p = base + row(16 * u + li);
      if constexpr (kWide) {
#pragma unroll
        for (int j = 0; j < KS / 2; ++j) {
          const u32x4 w = __builtin_nontemporal_load((const u32x4*)(p + 16 * (q + 4 * j)));
#pragma unroll
          for (int i = 0; i < 4; ++i) k[u][2 * j + i / 2][i % 2] = w[i];
        }
      } else {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          if constexpr (FMT == WMX_POOL_BF16) {
            const u32x4 w = __builtin_nontemporal_load((const u32x4*)(p + 16 * (q + 4 * s)));
#pragma unroll
            for (int i = 0; i < 4; ++i) k[u][s][i] = w[i];
          } else {
            const u32x2 w = __builtin_nontemporal_load((const u32x2*)(p + 8 * (q + 4 * s)));
            k[u][s][0] = w[0];
            k[u][s][1] = w[1];
          }
        }
      }
    }
  }
  template <class Row>
  __device__ __forceinline__ void load_v(const char* base, int li, int q, Row row) {
    typedef u32x4 u32x4_4 __attribute__((aligned(4)));
    typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));
    typedef u32x3 u32x3_4 __attribute__((aligned(4)));
    typedef u32x2 u32x2_4 __attribute__((aligned(4)));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const char* p = base + row(4 * q + (e & 3) + 16 * (e >> 2));
      if constexpr (FMT != WMX_POOL_BF16 && D == 96) {
        v[e][0] = __builtin_nontemporal_load((const uint32_t*)(p + 4 * li));
        v[e][1] = __builtin_nontemporal_load((const uint16_t*)(p + 64 + 2 * li));
      } else if constexpr (VD == 4) {
        const u32x4 w = __builtin_nontemporal_load((const u32x4_4*)(p + 16 * li));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[e][i] = w[i];
      } else if constexpr (VD == 3) {
        const u32x3 w = __builtin_nontemporal_load((const u32x3_4*)(p + 12 * li));
#pragma unroll
        for (int i = 0; i < 3; ++i) v[e][i] = w[i];
      } else if constexpr (VD == 2) {
        const u32x2 w = __builtin_nontemporal_load((const u32x2_4*)(p + 8 * li));
        v[e][0] = w[0];
        v[e][1] = w[1];
      } else {
        v[e][0] = __builtin_nontemporal_load((const uint32_t*)(p + 4 * li));
      }
    }
  }
  // MFMA operand of key half u, k-step s
  __device__ __forceinline__ u32x4 k_operand(int u, int s) const {
    if constexpr (FMT == WMX_POOL_BF16) {
      return u32x4{k[u][s][0], k[u][s][1], k[u][s][2], k[u][s][3]};
    } else {
      return u32x4{code_pair<FMT, false>(k[u][s][0]), code_pair<FMT, true>(k[u][s][0]), code_pair<FMT, false>(k[u][s][1]),
                   code_pair<FMT, true>(k[u][s][1])};
    }
  }
  // bf16 pair w (elements 2 w, 2 w + 1 of the lane's W) of key e
  __device__ __forceinline__ uint32_t v_pair(int e, int w) const {
    if constexpr (FMT == WMX_POOL_BF16) return v[e][w];
    else return w & 1 ? code_pair<FMT, true>(v[e][w / 2]) : code_pair<FMT, false>(v[e][w / 2]);
  }
};

struct TreeRange {
  int base;   // committed slots (every node sees them)
  int total;  // committed and drafted slots, within the pool
};

__device__ __forceinline__ TreeRange tree_range(const wmx_tree_args& a, int b) {
  int64_t len = a.kv_lengths ? a.kv_lengths[b] : a.kv_length_scalar;
  len = len < 0 ? 0 : len;
  const int64_t cap = a.capacity;
  int64_t base = len > cap ? cap : len + a.use_dummy;
  base = base > cap ? cap : base;
  const int64_t total = a.tree_mask ? min(base + a.nodes, cap) : base;
  return TreeRange{__builtin_amdgcn_readfirstlane((int)base), __builtin_amdgcn_readfirstlane((int)total)};
}

__device__ __forceinline__ float lane_from(float x, int lane) {
  return __uint_as_float(__builtin_amdgcn_ds_bpermute(lane << 2, __float_as_uint(x)));
}

template <int FMT, int D, int MB>
__global__ __launch_bounds__(64 * kTreeWaves, MB == 4 ? 1 : 2) void tree_kernel(const wmx_tree_args a, int units, int tiles,
                                                                          int nsplit, int chunk) {
  using Tile = TreeTile<FMT, D>;
  constexpr int KS = Tile::KS, W = Tile::W, ROWS = 16 * MB;
  constexpr int LDR = 4 * W + 4;  // LDS row of one merge round: four quarters x W, padded against bank conflicts
  __shared__ __attribute__((aligned(16))) float lds_o[kTreeWaves][ROWS][LDR];
  __shared__ float lds_m[kTreeWaves][ROWS], lds_l[kTreeWaves][ROWS];

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int li = lane & 15, q = lane >> 4;
  // blocks 8 apart share an XCD: the row tiles of one (range, row, KV head)
  // are placed so, and read its slots through one L2
  const int slab = blockIdx.x / (8 * tiles), in_slab = blockIdx.x - slab * 8 * tiles;
  const int unit = slab * 8 + (in_slab & 7), tile_row = in_slab >> 3;
  if (unit >= units) return;
  const int pairs = a.batch * a.kv_heads;
  const int split = unit / pairs, pair = unit - split * pairs;
  const int b = pair / a.kv_heads, hk = pair - b * a.kv_heads;
  const int group = a.q_heads / a.kv_heads;
  const int rows = a.nodes * group, row0 = tile_row * ROWS;

  const TreeRange range = tree_range(a, b);
  const int begin = split * chunk, end = min(begin + chunk, range.total);
  const float scale = a.softmax_scale * kLog2e;

  float m[MB], l[MB];
  f32x4 acc[MB][W];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    m[mb] = kNegInf;
    l[mb] = 0.f;
#pragma unroll
    for (int c = 0; c < W; ++c) acc[mb][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  if (begin < end) {
    // this lane's queries: rows row0 + 16 mb + li (zeros past the last)
    u32x4 qf[MB][KS];
    int node[MB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const int r = row0 + 16 * mb + li;
      const bool ok = r < rows;
      const int i = ok ? r / group : 0, h = hk * group + (ok ? r - i * group : 0);
      node[mb] = i;
      const bf16* p = (const bf16*)a.q + (int64_t)b * a.q_stride[0] + (int64_t)h * a.q_stride[1] + (int64_t)i * a.q_stride[2];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const u32x4 w = load16(p + Tile::k_dim(s, q));
        const u32x4 z = {0u, 0u, 0u, 0u};
        qf[mb][s] = ok ? w : z;
      }
    }
    const char* kbase = (const char*)a.k + ((int64_t)b * a.k_stride[0] + (int64_t)hk * a.k_stride[1]) * Tile::kElem;
    const char* vbase = (const char*)a.v + ((int64_t)b * a.v_stride[0] + (int64_t)hk * a.v_stride[1]) * Tile::kElem;
    const int64_t ksb = a.k_stride[2] * Tile::kElem, vsb = a.v_stride[2] * Tile::kElem;
    const float* kscale = FMT == WMX_POOL_BF16 ? nullptr : a.k_scales + (int64_t)b * a.k_scales_stride[0] + (int64_t)hk * a.k_scales_stride[1];
    const float* vscale = FMT == WMX_POOL_BF16 ? nullptr : a.v_scales + (int64_t)b * a.v_scales_stride[0] + (int64_t)hk * a.v_scales_stride[1];
    const uint8_t* kmask = a.key_mask ? a.key_mask + (int64_t)b * a.key_mask_stride : nullptr;
    const uint8_t* tmask = a.tree_mask ? a.tree_mask + (int64_t)b * a.tree_mask_stride[0] : nullptr;
    const int ks32 = (int)ksb, vs32 = (int)vsb;  // a tile's rows span less than 2^31 bytes (checked on the host)

    Tile tile;
    float ks[8], vs[8];  // scales of the lane's keys
    const auto load_scales = [&](int j0, int last, const float* src, float (&out)[8]) {
      if constexpr (FMT != WMX_POOL_BF16) {
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = src[j0 + min(4 * q + (e & 3) + 16 * (e >> 2), last)];
      }
    };
    // rows past the last visible slot are read as the last one and masked
    const auto load_k = [&](int j0) {
      const int last = end - 1 - j0;
      tile.load_k(kbase + j0 * ksb, li, q, [&](int row) { return min(row, last) * ks32; });
      load_scales(j0, last, kscale, ks);
    };
    const auto load_v = [&](int j0) {
      const int last = end - 1 - j0;
      tile.load_v(vbase + j0 * vsb, li, q, [&](int row) { return min(row, last) * vs32; });
      load_scales(j0, last, vscale, vs);
    };

    int j0 = begin + kTreeTile * wave;
    if (j0 < end) {
      load_k(j0);
      load_v(j0);
    }
    for (; j0 < end; j0 += kTreeStep) {
      // S^T = K Q^T
      f32x4 s[MB][2];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) s[mb][0] = s[mb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < KS; ++st) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const u32x4 kf = tile.k_operand(u, st);
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) s[mb][u] = mfma16(kf, qf[mb][st], s[mb][u]);
        }
      }
      float sc[MB][8];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          sc[mb][e] = s[mb][e >> 2][e & 3] * (FMT == WMX_POOL_BF16 ? scale : scale * ks[e]);
      }
      const int next = j0 + kTreeStep;
      if (next < end) load_k(next);  // K's registers are free

      // slots that some row does not see: past the committed ones, or masked
      const bool edge = kmask || j0 + kTreeTile > min(range.base, end);
      uint32_t seen[MB];  // bit e: this lane's query sees its key e
      if (edge) {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) seen[mb] = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = j0 + 4 * q + (e & 3) + 16 * (e >> 2);
          bool ok = j < end;
          if (ok && kmask) ok = kmask[j] != 0;
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) {
            bool vis = ok;
            if (ok && j >= range.base) vis = tmask[(int64_t)node[mb] * a.tree_mask_stride[1] + (j - range.base)] != 0;
            seen[mb] |= (vis ? 1u : 0u) << e;
            sc[mb][e] = vis ? sc[mb][e] : kNegInf;
          }
        }
      }

      uint32_t p[MB][4];  // weights times V scales, the B operand
      float pf[MB][8];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        float top = sc[mb][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = fmaxf(top, sc[mb][e]);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        if (__any(top > m[mb])) {
          const float mn = fmaxf(m[mb], top);
          const float f = mn == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m[mb] - mn);
          l[mb] *= f;
#pragma unroll
          for (int c = 0; c < W; ++c) acc[mb][c] *= f;
          m[mb] = mn;
        }
        const float ref = m[mb] == kNegInf ? 0.f : m[mb];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float w = __builtin_amdgcn_exp2f(sc[mb][e] - ref);
          l[mb] += w;
          float x = w;
          if constexpr (FMT != WMX_POOL_BF16) {
            x = w * vs[e];
            if (edge) x = (seen[mb] >> e) & 1u ? x : 0.f;  // a masked row's scale may be NaN
          }
          pf[mb][e] = x;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) p[mb][i] = pack_bf16x2(pf[mb][2 * i], pf[mb][2 * i + 1]);
      }

      // O^T += V^T P^T, output blocks 2 w and 2 w + 1 at a time
      uint32_t odd = 0u;  // bit e: key e of this lane holds a value that is not finite
#pragma unroll
      for (int w = 0; w < W / 2; ++w) {
        uint32_t x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = tile.v_pair(e, w);
        if (FMT != WMX_POOL_INT8 && edge) {
          // A value that some row must not see may be anything: 0 times an
          // infinity is no zero, so such values leave the product and are
          // added below to the rows that see them.
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const bool lo = (x[e] & 0x7f80u) == 0x7f80u, hi = (x[e] & 0x7f800000u) == 0x7f800000u;
            odd |= (lo || hi ? 1u : 0u) << e;
            x[e] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
          }
        }
        u32x4 v0, v1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v0[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x05040100u);
          v1[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x07060302u);
        }
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          const u32x4 pb = {p[mb][0], p[mb][1], p[mb][2], p[mb][3]};
          acc[mb][2 * w] = mfma16(v0, pb, acc[mb][2 * w]);
          acc[mb][2 * w + 1] = mfma16(v1, pb, acc[mb][2 * w + 1]);
        }
      }
      if (FMT != WMX_POOL_INT8 && edge && __any(odd)) {
        // key by key: the weight from the lane that holds it, the values from
        // the lanes that loaded them
#pragma unroll 1
        for (int kq = 0; kq < 4; ++kq) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (!__any(q == kq && ((odd >> e) & 1u))) continue;
#pragma unroll
            for (int w = 0; w < W / 2; ++w) {
              const uint32_t pair_bits = tile.v_pair(e, w);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const uint32_t bits = (uint32_t)__builtin_amdgcn_ds_bpermute((16 * kq + 4 * q + r) << 2, (int)pair_bits);
#pragma unroll
                for (int mb = 0; mb < MB; ++mb) {
                  const float pw = lane_from(pf[mb][e], 16 * kq + li);
                  const bool vis = (__builtin_amdgcn_ds_bpermute((16 * kq + li) << 2, (int)seen[mb]) >> e) & 1;
                  const float lo = bf16_lo(bits), hi = bf16_hi(bits);
                  if (vis && (bits & 0x7f80u) == 0x7f80u) acc[mb][2 * w][r] += pw * lo;
                  if (vis && (bits & 0x7f800000u) == 0x7f800000u) acc[mb][2 * w + 1][r] += pw * hi;
                }
              }
            }
          }
        }
      }
      if (next < end) load_v(next);
    }
  }

  // the workgroup's waves merged: maxima and sums, then the outputs in four
  // rounds (round r: block rows 4 q + r, W consecutive d per lane)
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    l[mb] += __shfl_xor(l[mb], 16);
    l[mb] += __shfl_xor(l[mb], 32);
    if (q == 0) {
      lds_m[wave][16 * mb + li] = m[mb];
      lds_l[wave][16 * mb + li] = l[mb];
    }
  }
  __syncthreads();
  float* ws_o = (float*)a.workspace;
  float* ws_ml = ws_o + (int64_t)a.batch * a.q_heads * a.nodes * nsplit * D;
  const int64_t prow0 = ((int64_t)pair * rows + row0) * nsplit + split;  // partial of row row0; rows are nsplit apart
  const auto row_max = [&](int row) {
    float mx = lds_m[0][row];
#pragma unroll
    for (int w = 1; w < kTreeWaves; ++w) mx = fmaxf(mx, lds_m[w][row]);
    return mx;
  };
  const auto row_sum = [&](int row, float mx) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kTreeWaves; ++w)
      if (lds_m[w][row] != kNegInf || lds_l[w][row] != 0.f) sum += lds_l[w][row] * __builtin_amdgcn_exp2f(lds_m[w][row] - mx);
    return sum;
  };
  if (nsplit > 1 && tid < ROWS && row0 + tid < rows) {
    const float mx = row_max(tid);
    float* out = ws_ml + (prow0 + (int64_t)tid * nsplit) * 2;
    out[0] = mx;
    out[1] = row_sum(tid, mx == kNegInf ? 0.f : mx);
  }
  if (nsplit > 1 && begin >= end) return;  // (the workgroup agrees) its sum is zero: the merge skips it
  float factor[MB];  // this wave's share of its rows
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const float mx = row_max(16 * mb + li);
    factor[mb] = m[mb] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m[mb] - mx);
    if (m[mb] == kNegInf && l[mb] != 0.f) factor[mb] = 1.f;  // (a row of NaN scores)
  }
  constexpr int PAIRS = ROWS * 4 * W / 2;  // output pairs of a round
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    __syncthreads();
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
      for (int c = 0; c < W; c += 2) {
        float* dst = &lds_o[wave][16 * mb + li][W * q + c];
        dst[0] = acc[mb][c][r] * factor[mb];
        dst[1] = acc[mb][c + 1][r] * factor[mb];
      }
    }
    __syncthreads();
    for (int i = tid; i < PAIRS; i += 64 * kTreeWaves) {
      const int row = i / (2 * W), x = i - row * 2 * W;
      const int qq = x / (W / 2), c = 2 * (x - qq * (W / 2));
      if (row0 + row >= rows) continue;
      float o0 = 0.f, o1 = 0.f;
#pragma unroll
      for (int w = 0; w < kTreeWaves; ++w) {
        o0 += lds_o[w][row][W * qq + c];
        o1 += lds_o[w][row][W * qq + c + 1];
      }
      const int d = Tile::v_dim(4 * qq + r, c);  // (c even: d and d + 1)
      if (nsplit > 1) {
        float* out = ws_o + (prow0 + (int64_t)row * nsplit) * D + d;
        out[0] = o0;
        out[1] = o1;
      } else {
        const float mx = row_max(row), sum = row_sum(row, mx == kNegInf ? 0.f : mx);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int n = (row0 + row) / group, h = hk * group + (row0 + row - n * group);
        bf16* out = (bf16*)a.o + (int64_t)b * a.o_stride[0] + (int64_t)h * a.o_stride[1] + (int64_t)n * a.o_stride[2] + d;
        *(uint32_t*)out = pack_bf16x2(o0 * inv, o1 * inv);
      }
    }
  }
}

// Merge of a row's ranges: one thread per four consecutive d.
__global__ __launch_bounds__(256) void tree_merge_kernel(const wmx_tree_args a, int nsplit, int64_t threads) {
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (gid >= threads) return;
  const int D = a.head_dim, per = D / 4, group = a.q_heads / a.kv_heads, rows = a.nodes * group;
  const int64_t row = gid / per;
  const int d = 4 * (int)(gid - row * per);
  const float* ws_o = (const float*)a.workspace;
  const float* ws_ml = ws_o + (int64_t)a.batch * a.q_heads * a.nodes * nsplit * D + row * nsplit * 2;
  ws_o += row * nsplit * D + d;
  float mx = kNegInf;
  for (int s = 0; s < nsplit; ++s) mx = fmaxf(mx, ws_ml[2 * s]);
  const float ref = mx == kNegInf ? 0.f : mx;
  float sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < nsplit; ++s) {
    const float ls = ws_ml[2 * s + 1];
    if (ls == 0.f) continue;  // an empty range wrote no output
    const float ms = ws_ml[2 * s];
    const float w = ms == kNegInf ? 1.f : __builtin_amdgcn_exp2f(ms - ref);
    sum += ls * w;
    const f32x4 part = *(const f32x4*)(ws_o + (int64_t)s * D);
    o += part * w;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t pair = row / rows;
  const int in_pair = (int)(row - pair * rows), n = in_pair / group;
  const int b = (int)(pair / a.kv_heads), hk = (int)(pair - (int64_t)b * a.kv_heads), h = hk * group + in_pair - n * group;
  bf16* out = (bf16*)a.o + (int64_t)b * a.o_stride[0] + (int64_t)h * a.o_stride[1] + (int64_t)n * a.o_stride[2] + d;
  const u32x2 w = {pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
  typedef u32x2 u32x2_4 __attribute__((aligned(4)));
  *(u32x2_4*)out = w;
}

// Query rows per workgroup, in 16s.
static int tree_blocks(const wmx_tree_args& a) {
  const int64_t rows = (int64_t)a.nodes * (a.q_heads / a.kv_heads);
  return rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
}
static int64_t tree_tiles(const wmx_tree_args& a) {
  const int64_t rows = (int64_t)a.nodes * (a.q_heads / a.kv_heads), per = 16 * tree_blocks(a);
  return (rows + per - 1) / per;
}

int tree_num_splits(const wmx_tree_args& a) {
  if (a.num_splits > 0) return a.num_splits;
  const int64_t wgs = (int64_t)a.batch * a.kv_heads * tree_tiles(a);
  if (wgs <= 0) return 1;
  int64_t splits = (4 * 256 + wgs - 1) / wgs;
  const int64_t most = ((int64_t)a.capacity + 2 * kTreeStep - 1) / (2 * kTreeStep);
  if (splits > most) splits = most;
  return splits < 1 ? 1 : (int)splits;
}

int64_t tree_workspace_size(const wmx_tree_args& a) {
  const int64_t s = tree_num_splits(a);
  return s == 1 ? 0 : (int64_t)a.batch * a.q_heads * a.nodes * s * (a.head_dim + 2) * (int64_t)sizeof(float);
}

template <int FMT, int D>
static void launch_tree_d(const wmx_tree_args& a, unsigned blocks, int units, int tiles, int nsplit, int chunk, hipStream_t stream) {
  const dim3 grid(blocks), block(64 * kTreeWaves);
  switch (tree_blocks(a)) {
    case 1: hipLaunchKernelGGL((tree_kernel<FMT, D, 1>), grid, block, 0, stream, a, units, tiles, nsplit, chunk); break;
    case 2: hipLaunchKernelGGL((tree_kernel<FMT, D, 2>), grid, block, 0, stream, a, units, tiles, nsplit, chunk); break;
    default: hipLaunchKernelGGL((tree_kernel<FMT, D, 4>), grid, block, 0, stream, a, units, tiles, nsplit, chunk); break;
  }
}

template <int FMT>
static int launch_tree_f(const wmx_tree_args& a, unsigned blocks, int units, int tiles, int nsplit, int chunk, hipStream_t stream) {
  switch (a.head_dim) {
    case 64: launch_tree_d<FMT, 64>(a, blocks, units, tiles, nsplit, chunk, stream); return WMX_OK;
    case 96: launch_tree_d<FMT, 96>(a, blocks, units, tiles, nsplit, chunk, stream); return WMX_OK;
    case 128: launch_tree_d<FMT, 128>(a, blocks, units, tiles, nsplit, chunk, stream); return WMX_OK;
    default: return WMX_E_UNSUPPORTED;
  }
}

int launch_tree(const wmx_tree_args& a, hipStream_t stream) {
  const int nsplit = tree_num_splits(a);
  const int64_t units = (int64_t)nsplit * a.batch * a.kv_heads, tiles = tree_tiles(a);
  const int64_t blocks = (units + 7) / 8 * 8 * tiles;
  const int64_t merged = (int64_t)a.batch * a.q_heads * a.nodes * (a.head_dim / 4);
  if (blocks > INT32_MAX || (merged + 255) / 256 > INT32_MAX) return WMX_E_UNSUPPORTED;
  int64_t chunk = ((int64_t)a.capacity + nsplit - 1) / nsplit;
  chunk = (chunk + kTreeStep - 1) / kTreeStep * kTreeStep;
  if (chunk < kTreeStep) chunk = kTreeStep;
  if (chunk * nsplit > INT32_MAX) return WMX_E_UNSUPPORTED;  // (ranges begin within 31 bits)
  int rc;
  if (a.format == WMX_POOL_BF16) rc = launch_tree_f<WMX_POOL_BF16>(a, (unsigned)blocks, (int)units, (int)tiles, nsplit, (int)chunk, stream);
  else if (a.format == WMX_POOL_E4M3) rc = launch_tree_f<WMX_POOL_E4M3>(a, (unsigned)blocks, (int)units, (int)tiles, nsplit, (int)chunk, stream);
  else rc = launch_tree_f<WMX_POOL_INT8>(a, (unsigned)blocks, (int)units, (int)tiles, nsplit, (int)chunk, stream);
  if (rc != WMX_OK || nsplit == 1) return rc;
  hipLaunchKernelGGL(tree_merge_kernel, dim3((unsigned)((merged + 255) / 256)), dim3(256), 0, stream, a, nsplit, merged);
  return WMX_OK;
}

}  // namespace wmx
