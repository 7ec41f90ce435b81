// Attention of drafted tokens (a tree, or one token) over a bf16 or quantised
// KV pool for gfx950 (visibility and formats in wmx_attn.h).
//
// The query rows of one KV head (nodes x query heads of its group, node-major)
// share its keys and values, so a workgroup takes 16 MB of them and a range of
// slots; each K/V byte is read from HBM once per row tile and converted once.
// Four waves (eight where there are few workgroups) take turns at the range's
// 32-slot tiles and keep their own running maximum, sum and output, merged
// through LDS at the end; ranges of one row are merged by a second kernel in
// log-sum-exp form.
//
// With v_mfma_f32_16x16x32_bf16
//   S^T = K Q^T    A: lane l holds key l % 16, 8 consecutive d of its quarter
//                  l / 16; the d order is the one in which its reads are
//                  widest, the same for Q. K tiles pass through LDS (see
//                  k_swizzle), and the scales with them
//   O^T = V^T P^T  B: P as S^T left it in the accumulators: lane (query l % 16,
//                  quarter q) holds keys 4 q + [0, 4) of the tile's two
//                  16-key halves; A: V of those keys, loaded as D/16
//                  consecutive d per lane and transposed between registers
//                  (v_perm), so output block c holds d = (D/16) i + c
// K and V scales multiply scores and weights, one operation per score instead
// of one per element. Codes are converted exactly: K's to bf16 like the
// queries; V's to fp16, in which the weights keep 11 bits (bf16 pools: 8).
#include <climits>
#include "lds_tiles.h"
#include "wmx_kernels.h"

namespace wmx {

// The running maximum follows a larger score only once it is past it by this
// many powers of two: weights up to 2^8 cost no precision, and most steps
// rescale nothing.
constexpr float kLazyMax = 8.f;
// V scales times 2^lv stay at most 64, so that weights times scales stay below
// 2^14 in fp16 (largest 65,504). Its smallest step is 2^-24: a weight of one takes
// its full bits on scales down to 2^-20 of the largest, and an error of 2^-31 of the
// largest is the most there is below.
constexpr float kScaleRoom = 64.f;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Two codes (the low or high half of a dword) as a bf16 or fp16 pair, exactly.
template <int FMT, bool HIGH>
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  if constexpr (FMT == WMX_POOL_E4M3) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
  } else {
    const int s = HIGH ? 16 : 0;
    return pack_bf16x2((float)(int8_t)(w >> s), (float)(int8_t)(w >> (s + 8)));
  }
}
template <int FMT, bool HIGH>
__device__ __forceinline__ uint32_t code_pair_half(uint32_t w) {
  if constexpr (FMT == WMX_POOL_E4M3) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HIGH));
  } else {
    // 1024 + (code + 128) has the code's bits as its lowest: no conversion
    const uint32_t biased = __builtin_amdgcn_perm(0x64646464u, w ^ 0x80808080u, HIGH ? 0x04030402u : 0x04010400u);
    const f16x2 x = __builtin_bit_cast(f16x2, biased) - f16x2{(_Float16)1152.f, (_Float16)1152.f};
    return __builtin_bit_cast(uint32_t, x);
  }
}

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

// The weights of a query row are x = exp2(t - ref), t its scaled scores in powers
// of two and ref = m - lv: m a score near the largest so far, 2^lv a factor that
// keeps weights times V scales within fp16 (0 for bf16 pools). Sums and outputs
// hold x and its products; `limit` is the t - ref from which ref moves: lv +
// kLazyMax, or -inf until the row has seen a slot.
struct TreeRow {
  float ref, limit, l;

  __device__ __forceinline__ void start(float lv) {
    ref = -lv;
    limit = kNegInf;
    l = 0.f;
  }
  // For lanes of rows with a score past their limit (top: the row's largest t -
  // ref): how far ref moves, and the factor that sums and outputs take.
  __device__ __forceinline__ float move(float top, float lv, float& factor) {
    const bool seen = limit != kNegInf;
    float up = top - lv;
    up = seen ? fmaxf(up, 0.f) : top == kNegInf ? 0.f : up;
    factor = seen ? __builtin_amdgcn_exp2f(-up) : 1.f;  // (nothing to scale before the first slot)
    ref += up;
    l *= factor;
    limit = seen || top > kNegInf ? lv + kLazyMax : kNegInf;
    return up;
  }
  // Another lv, `by` larger; `factor` = 2^by.
  __device__ __forceinline__ void rescale(float by, float factor) {
    ref -= by;
    limit += by;
    l *= factor;
  }
  // The maximum that goes with l / 2^lv.
  __device__ __forceinline__ float max_score(float lv) const { return limit == kNegInf ? kNegInf : ref + lv; }
};

// The lv that takes the largest V scale `most` of a tile (over the wave) into
// [32, 64) for the weight 1, and the one to begin with: any but the smallest
// scales replace it, and sums of 2^lv stay finite.
__device__ __forceinline__ float scale_lv(float most) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) most = fmaxf(most, __shfl_xor(most, o));
  return (float)min(132 - (int)(__float_as_uint(most) >> 23), 100);
}
constexpr float kScaleStart = 100.f;

constexpr int kTreeTile = 32;                      // slots per wave and step

__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16_half(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// How a wave reads 32 slots of K and V.
template <int FMT, int D, int MB>
struct TreeTile {
  // cache policy: nontemporal for slots read once; with two row blocks other row
  // tiles, on the same XCD, read them too (64 nodes over 16 x 8,192 slots of e4m3:
  // 102 us, 114 nontemporal; one token over 32 such rows 68 and 63)
  static constexpr int kPolicy = MB == 1 ? 2 : 0;
  static constexpr int kElem = FMT == WMX_POOL_BF16 ? 2 : 1;  // bytes
  static constexpr int kRow = D * kElem;
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
  // the lane's key e of a tile
  static __device__ __forceinline__ int key_of(int q, int e) { return 4 * q + (e & 3) + 16 * (e >> 2); }

  uint32_t k[2][KS][KD];  // key halves
  uint32_t v[8][VD];      // the lane's keys

  // K goes through LDS: lanes next to each other load chunks of 16 bytes next to
  // each other, which the L1 serves a line at a time, where the operand's lanes
  // are rows, and 64 lines an instruction (64 nodes over 16 rows of up to 8,192
  // slots: 86 us, 102 with the operands loaded directly). Chunk c of row r is
  // stored as chunk c ^ k_swizzle(r) (D = 96 by pairs or fours), so that 16 rows'
  // chunks c lie in different banks.
  static constexpr int kChunks = kRow / 16, kLoads = kTreeTile * kChunks / 64;
  static __device__ __forceinline__ int k_swizzle(int r) {
    if constexpr (kRow == 192) return (r >> 2) & 3;
    else if constexpr (kRow == 96) return (r >> 3) & 1;
    else return (r / (256 / kRow)) & (kChunks - 1);
  }
  // byte offset of what lane `lane` loads with instruction i
  static __device__ __forceinline__ int k_source(int lane, int i, int step) {
    const int g = 64 * i + lane, r = g / kChunks;
    return r * step + 16 * ((g - r * kChunks) ^ k_swizzle(r));
  }
  static __device__ __forceinline__ void stage_k(const rsrc_t& rs, char* stage, const int (&off)[kLoads]) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(stage + 1024 * i), 16, off[i], 0, 0, kPolicy);
  }
  __device__ __forceinline__ void read_k(const char* stage, int li, int q) {
    const int swz = k_swizzle(li);  // (rows 16 apart share it)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const char* row = stage + (16 * u + li) * kRow;
      if constexpr (kWide) {
#pragma unroll
        for (int j = 0; j < KS / 2; ++j) {
          const u32x4 w = *(const u32x4*)(row + 16 * ((q + 4 * j) ^ swz));
#pragma unroll
          for (int i = 0; i < 4; ++i) k[u][2 * j + i / 2][i % 2] = w[i];
        }
      } else {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          if constexpr (FMT == WMX_POOL_BF16) {
            const u32x4 w = *(const u32x4*)(row + 16 * ((q + 4 * s) ^ swz));
#pragma unroll
            for (int i = 0; i < 4; ++i) k[u][s][i] = w[i];
          } else {
            const u32x2 w = *(const u32x2*)(row + 16 * (((q >> 1) + 2 * s) ^ swz) + 8 * (q & 1));
            k[u][s][0] = w[0];
            k[u][s][1] = w[1];
          }
        }
      }
    }
  }

  __device__ __forceinline__ void load_v(const rsrc_t& rs, const int (&off)[8], int li) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (FMT != WMX_POOL_BF16 && D == 96) {
        v[e][0] = __builtin_amdgcn_raw_buffer_load_b32(rs, off[e], 0, kPolicy);
        v[e][1] = __builtin_amdgcn_raw_buffer_load_b16(rs, off[e] + 64 - 2 * li, 0, kPolicy);
      } else if constexpr (VD == 4) {
        const auto w = __builtin_amdgcn_raw_buffer_load_b128(rs, off[e], 0, kPolicy);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[e][i] = w[i];
      } else if constexpr (VD == 3) {
        const auto w = __builtin_amdgcn_raw_buffer_load_b96(rs, off[e], 0, kPolicy);
#pragma unroll
        for (int i = 0; i < 3; ++i) v[e][i] = w[i];
      } else if constexpr (VD == 2) {
        const auto w = __builtin_amdgcn_raw_buffer_load_b64(rs, off[e], 0, kPolicy);
        v[e][0] = w[0];
        v[e][1] = w[1];
      } else {
        v[e][0] = __builtin_amdgcn_raw_buffer_load_b32(rs, off[e], 0, kPolicy);
      }
    }
  }
  // byte offset of the lane's V part in a row (its first part, D = 96 codes)
  static __device__ __forceinline__ int v_part(int li) { return FMT != WMX_POOL_BF16 && D == 96 ? 4 * li : W * kElem * li; }

  // MFMA operand of key half u, k-step s
  __device__ __forceinline__ u32x4 k_operand(int u, int s) const {
    if constexpr (FMT == WMX_POOL_BF16) {
      return u32x4{k[u][s][0], k[u][s][1], k[u][s][2], k[u][s][3]};
    } else {
      return u32x4{code_pair<FMT, false>(k[u][s][0]), code_pair<FMT, true>(k[u][s][0]), code_pair<FMT, false>(k[u][s][1]),
                   code_pair<FMT, true>(k[u][s][1])};
    }
  }
  // pair w (elements 2 w, 2 w + 1 of the lane's W) of key e: bf16, or fp16 of codes
  __device__ __forceinline__ uint32_t v_pair(int e, int w) const {
    if constexpr (FMT == WMX_POOL_BF16) return v[e][w];
    else return w & 1 ? code_pair_half<FMT, true>(v[e][w / 2]) : code_pair_half<FMT, false>(v[e][w / 2]);
  }
  // exponent bits of a value that is not finite, in a v_pair's low half
  static constexpr uint32_t kOdd = FMT == WMX_POOL_BF16 ? 0x7f80u : 0x7c00u;
};

// Steps of a batch row, per KV head (one at least: its outputs are written).
__device__ __forceinline__ int tree_steps(const wmx_tree_args& a, int b, int step) {
  int64_t len = a.kv_lengths ? a.kv_lengths[b] : a.kv_length_scalar;
  len = len < 0 ? 0 : len > a.capacity ? a.capacity : len + a.use_dummy;
  const int64_t total = min(a.tree_mask ? len + a.nodes : len, (int64_t)a.capacity);
  return max(1, (int)((total + step - 1) / step));
}

// x of lanes l ^ 16 and l ^ 32 joined with this lane's, the same in all four
__device__ __forceinline__ float max_quarters(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return max_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_quarters(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return sum_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// One wave's state over its tiles, every NW-th of its workgroup's.
template <int FMT, int D, int MB, int NW>
struct TreeWave {
  using Tile = TreeTile<FMT, D, MB>;
  static constexpr int KS = Tile::KS, W = Tile::W;

  u32x4 qf[MB][KS];  // queries, the B operand
  TreeRow row[MB];
  f32x4 acc[MB][W];
  float lv, vref;    // (vref = 2^lv)
  Tile tile;
  float ks[8], vs[8];
  int koff[Tile::kLoads], voff[8];
  char* stage;       // this wave's K tile in LDS, and behind it the K and V scales of its slots
  uint32_t kept[8];  // key_mask of the lane's keys
  bool odd;          // this lane met a drafted value that is not finite

  // of the whole wave
  const char *kbase, *vbase;
  const float *kscale, *vscale;
  const uint8_t *kmask, *tmask;
  int node_at[MB];                   // offset of this lane's node's row in tmask
  int tree_bytes;
  int64_t ksb, vsb;                  // bytes between slots
  int base, end;
  float scale;

  // bytes of up to a tile's rows
  static __device__ __forceinline__ int span(int slots, int64_t step) {
    return slots > 0 ? (int)((min(slots, kTreeTile) - 1) * step) + Tile::kRow : 0;
  }
  static constexpr int kTileBytes = kTreeTile * Tile::kRow;
  // 32 K scales, 32 V scales: half the lanes load zeros past them
  __device__ __forceinline__ void stage_scales(int j0, int lane) {
    if constexpr (FMT != WMX_POOL_BF16) {
      const int bytes = 4 * max(0, min(end - j0, kTreeTile));
      __builtin_amdgcn_raw_ptr_buffer_load_lds(make_rsrc(kscale + j0, bytes), (lds_void*)(stage + kTileBytes), 4, 4 * lane, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(make_rsrc(vscale + j0, bytes), (lds_void*)(stage + kTileBytes + 256), 4, 4 * lane, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void read_scales(int q) {
    if constexpr (FMT != WMX_POOL_BF16) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const f32x4 a = *(const f32x4*)(stage + kTileBytes + 16 * q + 64 * u), b = *(const f32x4*)(stage + kTileBytes + 256 + 16 * q + 64 * u);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ks[4 * u + i] = a[i];
          vs[4 * u + i] = b[i];
        }
      }
    }
  }
  // Slots past the last visible one read as zeros, and so does a tile past it: the
  // loads of the next tile are issued without a branch around them, whose other
  // side would make the waits for K wait for V as well.
  template <bool EDGE>
  __device__ __forceinline__ void load_k(int j0, int lane, int q) {
    Tile::stage_k(make_rsrc(kbase + j0 * ksb, span(end - j0, ksb)), stage, koff);
    stage_scales(j0, lane);
    if (EDGE && kmask) {  // (zero past the last slot; with a key mask every tile is an edge)
      const rsrc_t rs = make_rsrc(kmask, end);
#pragma unroll
      for (int e = 0; e < 8; ++e) kept[e] = __builtin_amdgcn_raw_buffer_load_b8(rs, j0 + Tile::key_of(q, e), 0, 0);
    }
  }
  __device__ __forceinline__ void load_v(int j0, int q, int li) {
    tile.load_v(make_rsrc(vbase + j0 * vsb, span(end - j0, vsb)), voff, li);
  }

  // One tile. EDGE: some of its slots are masked, drafted or past the end.
  template <bool EDGE>
  __device__ __forceinline__ void step(int j0, int li, int q) {
    uint32_t seen[MB];      // bit e: this lane's query sees its key e
    uint32_t keep[8];       // 0: no query may see key e, else all ones
    uint32_t drafted = 0u;  // bit e: key e is a drafted one
    const bool any_drafted = EDGE && j0 + kTreeTile > base && end > base;
    if constexpr (EDGE) {
      uint32_t kept_bits = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = j0 + Tile::key_of(q, e);
        const bool ok = j < end && (!kmask || kept[e] != 0);
        keep[e] = ok ? ~0u : 0u;
        opaque(keep[e]);
        kept_bits |= (ok ? 1u : 0u) << e;
        drafted |= (ok && j >= base ? 1u : 0u) << e;
      }
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) seen[mb] = kept_bits;
      if (any_drafted) {
        // (a query's bytes past the last slot and before the first drafted one are not read)
        const rsrc_t rs = make_rsrc(tmask, tree_bytes);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          uint32_t t[8];
          opaque(drafted);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int a = j0 + Tile::key_of(q, e) - base;
            t[e] = __builtin_amdgcn_raw_buffer_load_b8(rs, (drafted >> e) & 1u ? node_at[mb] + a : -1, 0, 0);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) seen[mb] &= ~((t[e] ? 0u : (drafted >> e) & 1u) << e);
        }
      }
    }
    // K and the scales go to registers, and the next tile's into their place
    const int next = j0 + NW * kTreeTile, lane = 16 * q + li;
    tile.read_k(stage, li, q);
    read_scales(q);
    lgkm_settle();
    load_k<EDGE>(next, lane, q);

    float sc[MB][8];
    {
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
      // scores over the reference: the weights are exp2 of them
      float kq[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) kq[e] = FMT == WMX_POOL_BF16 ? scale : scale * ks[e];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sc[mb][e] = fmaf(s[mb][e >> 2][e & 3], kq[e], -row[mb].ref);
      }
    }

    if constexpr (EDGE) {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        opaque(seen[mb]);
#pragma unroll
        for (int e = 0; e < 8; ++e) sc[mb][e] = (seen[mb] >> e) & 1u ? sc[mb][e] : kNegInf;
      }
    }

    if constexpr (FMT != WMX_POOL_BF16) {
      float most = 0.f;  // (NaN stays out of it)
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(vs[e]));
      if (__any(most * vref > kScaleRoom)) {
        most = 0.f;  // (and here an infinity)
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(vs[e]) < kPosInf ? fabsf(vs[e]) : 0.f);
        const float to = scale_lv(most), f = __builtin_amdgcn_exp2f(to - lv);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          row[mb].rescale(to - lv, f);
#pragma unroll
          for (int c = 0; c < W; ++c) acc[mb][c] *= f;
#pragma unroll
          for (int e = 0; e < 8; ++e) sc[mb][e] += to - lv;
        }
        lv = to;
        vref = __builtin_amdgcn_exp2f(lv);
      }
    }

    u32x4 p[MB];  // weights (times V scales), the B operand
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      float top = fmaxf(sc[mb][0], sc[mb][1]);
#pragma unroll
      for (int e = 2; e < 8; ++e) top = fmaxf(top, sc[mb][e]);
      if (__any(top > row[mb].limit)) {
        float f;
        const float up = row[mb].move(max_quarters(top), lv, f);
#pragma unroll
        for (int c = 0; c < W; ++c) acc[mb][c] *= f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sc[mb][e] -= up;
      }
      float x[8];
      if constexpr (EDGE) opaque(seen[mb]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = __builtin_amdgcn_exp2f(sc[mb][e]);
        row[mb].l += x[e];
        if constexpr (FMT != WMX_POOL_BF16) {
          x[e] *= vs[e];
          if constexpr (EDGE) x[e] = (seen[mb] >> e) & 1u ? x[e] : 0.f;  // a masked row's scale may be NaN
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (FMT == WMX_POOL_BF16) {
          p[mb][i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
        } else {
          const f16x2 h = {(_Float16)x[2 * i], (_Float16)x[2 * i + 1]};
          p[mb][i] = __builtin_bit_cast(uint32_t, h);
        }
      }
    }

    // O^T += V^T P^T, output blocks 2 w and 2 w + 1 at a time
#pragma unroll
    for (int w = 0; w < W / 2; ++w) {
      uint32_t x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = tile.v_pair(e, w);
      if constexpr (EDGE && FMT != WMX_POOL_INT8) {
        // Zero times an infinity is no zero: masked rows leave the product, and
        // so do the values of drafted rows that are not finite, since some
        // queries do not see them (the others get them with the output).
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] &= keep[e];
        if (any_drafted) {
          opaque(drafted);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const bool draft = (drafted >> e) & 1u;
            const bool lo = draft && (x[e] & Tile::kOdd) == Tile::kOdd;
            const bool hi = draft && (x[e] & (Tile::kOdd << 16)) == Tile::kOdd << 16;
            odd |= lo || hi;
            x[e] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
          }
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
        if constexpr (FMT == WMX_POOL_BF16) {
          acc[mb][2 * w] = mfma16(v0, p[mb], acc[mb][2 * w]);
          acc[mb][2 * w + 1] = mfma16(v1, p[mb], acc[mb][2 * w + 1]);
        } else {
          acc[mb][2 * w] = mfma16_half(v0, p[mb], acc[mb][2 * w]);
          acc[mb][2 * w + 1] = mfma16_half(v1, p[mb], acc[mb][2 * w + 1]);
        }
      }
    }
    load_v(next, q, li);
  }
};

// Which key range a workgroup takes. The slots of every (batch row, KV head), the
// drafted ones included, are counted in steps of a workgroup (32 per wave). With
// nsplit 0 the workgroups are dealt out by these counts: all steps over `share`
// workgroups give a part, a (row, head) of n steps gets ceil(n / part) workgroups,
// and these split its steps evenly; a row of one writes the outputs itself. Rows
// of any lengths then load the card alike, whatever the pool's capacity. With
// nsplit > 0 every (row, head) has that many ranges of `share` steps.
struct TreeLaunch {
  int tiles, ranges, nsplit, share, waves;
};
// One range a row, in one launch, for pools of up to so many slots, and of twice
// as many where the rows' workgroups fill the CUs: the second launch, the partials
// and the dealing cost more than idle CUs do. Up to a workgroup a CU, eight waves
// share the row's slots. Us, one range and dealt, e4m3, 8 KV heads of two queries:
// 1,153 slots, one token over one row (D 64) 9 and 13; 1,700 slots (D 128) one row
// 11 and 14, 8 rows 15 and 17, 64 nodes over 8 rows 22 and 30; 2,500 slots, 4
// rows 17 and 17, 8 rows 20 and 17.5, 32 rows 23.5 and 30. 3,500 slots, 4 rows 22
// and 17, but 32 rows 30 and 35, 16 nodes 32 and 42; 4,800 slots, 32 rows 36 and
// 38.5. Eight waves and four: 16 nodes over 8 rows of 1,280 slots 17.3 and 19.1,
// with more than a workgroup a CU 64 nodes over 32 rows of 1,700 slots 70 and 54.
constexpr int kOneRange = 2560, kCUs = 256;
constexpr int kPlanRows = 256;  // most batch rows whose workgroups are dealt out
// How the steps are dealt, by the query rows of a workgroup: 16 rows stream the
// slots, and four workgroups a CU, of at least four steps, are best (e4m3, D 128,
// 8 KV heads, up to 8,192 slots, one token: 32 rows 58.5 us, 60 with two a CU, 61
// with eight; 8 rows 24 us, 29 with workgroups of two steps). With 32 rows the
// arithmetic sets the pace: one a CU, of any length (64 nodes over 16 such rows 85
// us, 92 with two a CU; 13 nodes over 4 bf16 rows of 4,096 slots 21, 23, with
// four a CU 29).
__host__ __device__ constexpr int tree_dealt(int rows) { return rows == 16 ? 1024 : 256; }
__host__ __device__ constexpr int tree_min_share(int rows) { return rows == 16 ? 4 : 1; }
// At the workspace's start, for the merge: the ranges before each row (per KV head), and all.
constexpr int kPlanInts = 512;
struct TreePartials {
  float *ml, *o;
};
__host__ __device__ inline int64_t tree_partial_rows(const TreeLaunch& t, int rows) {
  return (int64_t)t.ranges * t.tiles * rows;
}
__device__ __forceinline__ TreePartials tree_partials(const wmx_tree_args& a, const TreeLaunch& t, int rows) {
  float* o = (float*)a.workspace + kPlanInts;
  return TreePartials{o + tree_partial_rows(t, rows) * a.head_dim, o};
}

template <int FMT, int D, int MB, int NW>
__global__ __launch_bounds__(64 * NW, (NW == 4 && MB == 1 && TreeTile<FMT, D, MB>::kRow < 256) ? 3 : 2) void tree_kernel(
    const wmx_tree_args a, const TreeLaunch t) {
  using Tile = TreeTile<FMT, D, MB>;
  constexpr int KS = Tile::KS, W = Tile::W, ROWS = 16 * MB, STEP = NW * kTreeTile;
  constexpr int LDR = 4 * W + 4;  // LDS row of one merge round: four quarters x W, padded against bank conflicts
  __shared__ __attribute__((aligned(16))) float lds_o[NW][ROWS][LDR];
  __shared__ __attribute__((aligned(16))) char stage[NW][TreeWave<FMT, D, MB, NW>::kTileBytes + (FMT == WMX_POOL_BF16 ? 0 : 512)];
  __shared__ float lds_m[NW][ROWS], lds_l[NW][ROWS], lds_max[ROWS], lds_sum[ROWS];
  __shared__ int lds_odd, lds_wave[NW], lds_all[NW], lds_first[4];

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int li = lane & 15, q = lane >> 4;
  // blocks 8 apart share an XCD: the row tiles of one range are placed so, and
  // read its slots through one L2
  const int slab = blockIdx.x / (8 * t.tiles), in_slab = blockIdx.x - slab * 8 * t.tiles;
  const int index = slab * 8 + (in_slab & 7), tile_row = in_slab >> 3;  // of the range, of the row tile
  if (index >= t.ranges) return;
  const int group = a.q_heads / a.kv_heads;
  const int rows = a.nodes * group, row0 = tile_row * ROWS;

  // ---- the range: steps [s0, s1) of (b, hk) ----
  int b, hk, s0, s1, parts;
  if (t.nsplit > 0) {
    const int unit = index / t.nsplit;
    b = unit / a.kv_heads;
    hk = unit - b * a.kv_heads;
    s0 = (index - unit * t.nsplit) * t.share;
    s1 = s0 + t.share;
    parts = t.nsplit;
  } else {
    const int steps = tid < a.batch ? tree_steps(a, tid, STEP) : 0;
    int sum = steps;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) lds_wave[wave] = sum;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) all += lds_wave[i];
    const int share = max(tree_min_share(ROWS), (all * a.kv_heads + t.share - 1) / t.share);
    const int n = (steps + share - 1) / share;
    int before = n;  // inclusive scan over the workgroup
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(before, o);
      before += lane >= o ? up : 0;
    }
    if (lane == 63) lds_all[wave] = before;
    __syncthreads();
    int ranges = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      before += i < wave ? lds_all[i] : 0;
      ranges += lds_all[i];
    }
    before -= n;
    if (index == 0 && tile_row == 0) {
      int* plan = (int*)a.workspace;
      if (tid < a.batch) plan[tid] = before;
      if (tid == 0) plan[a.batch] = ranges;
    }
    if (index >= ranges * a.kv_heads) return;
    if (index >= before * a.kv_heads && index < (before + n) * a.kv_heads) {
      lds_first[0] = tid;
      lds_first[1] = index - before * a.kv_heads;
      lds_first[2] = n;
      lds_first[3] = steps;
    }
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(lds_first[0]);
    const int at = __builtin_amdgcn_readfirstlane(lds_first[1]), total = __builtin_amdgcn_readfirstlane(lds_first[3]);
    parts = __builtin_amdgcn_readfirstlane(lds_first[2]);
    hk = at / parts;
    const int part = at - hk * parts, each = total / parts, more = total - each * parts;
    s0 = part * each + min(part, more);
    s1 = s0 + each + (part < more);
  }
  const TreeRange range = tree_range(a, b);
  const bool complete = parts == 1;
  const int begin = min(s0 * STEP, range.total), end = min(s1 * STEP, range.total);
  const uint8_t* kmask = a.key_mask ? a.key_mask + (int64_t)b * a.key_mask_stride : nullptr;
  const uint8_t* tmask = a.tree_mask ? a.tree_mask + (int64_t)b * a.tree_mask_stride[0] : nullptr;
  const char* vbase = (const char*)a.v + ((int64_t)b * a.v_stride[0] + (int64_t)hk * a.v_stride[1]) * Tile::kElem;
  const int64_t vsb = a.v_stride[2] * Tile::kElem;
  if (tid == 0) lds_odd = 0;

  TreeWave<FMT, D, MB, NW> w;
  w.lv = FMT == WMX_POOL_BF16 ? 0.f : kScaleStart;
  w.vref = __builtin_amdgcn_exp2f(w.lv);
  w.odd = false;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    w.row[mb].start(w.lv);
#pragma unroll
    for (int c = 0; c < W; ++c) w.acc[mb][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  int j0 = begin + kTreeTile * wave;
  if (j0 < end) {
    w.kbase = (const char*)a.k + ((int64_t)b * a.k_stride[0] + (int64_t)hk * a.k_stride[1]) * Tile::kElem;
    w.vbase = vbase;
    w.ksb = a.k_stride[2] * Tile::kElem;
    w.vsb = vsb;
    if constexpr (FMT != WMX_POOL_BF16) {
      w.kscale = a.k_scales + (int64_t)b * a.k_scales_stride[0] + (int64_t)hk * a.k_scales_stride[1];
      w.vscale = a.v_scales + (int64_t)b * a.v_scales_stride[0] + (int64_t)hk * a.v_scales_stride[1];
    }
    w.kmask = kmask;
    w.tmask = tmask;
    w.tree_bytes = (int)((a.nodes - 1) * a.tree_mask_stride[1]) + a.nodes;
    w.base = range.base;
    w.end = end;
    w.scale = a.softmax_scale * kLog2e;
#pragma unroll
    for (int i = 0; i < Tile::kLoads; ++i) w.koff[i] = Tile::k_source(lane, i, (int)w.ksb);
    w.stage = stage[wave];
#pragma unroll
    for (int e = 0; e < 8; ++e) w.voff[e] = Tile::key_of(q, e) * (int)vsb + Tile::v_part(li);
    w.template load_k<true>(j0, lane, q);
    w.load_v(j0, q, li);
    // this lane's queries: rows row0 + 16 mb + li (zeros past the last)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const int r = row0 + 16 * mb + li;
      const bool ok = r < rows;
      const int i = ok ? r / group : 0, h = hk * group + (ok ? r - i * group : 0);
      w.node_at[mb] = i * (int)a.tree_mask_stride[1];
      const bf16* p = (const bf16*)a.q + (int64_t)b * a.q_stride[0] + (int64_t)h * a.q_stride[1] + (int64_t)i * a.q_stride[2];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const u32x4 x = load16(p + Tile::k_dim(s, q));
        const u32x4 z = {0u, 0u, 0u, 0u};
        w.qf[mb][s] = ok ? x : z;
      }
    }
    const int whole = kmask ? begin : min(range.base, end);  // slots that every query sees end here
    for (; j0 + kTreeTile <= whole; j0 += STEP) w.template step<false>(j0, li, q);
    for (; j0 < end; j0 += STEP) w.template step<true>(j0, li, q);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the last loads into LDS (zeros, of a tile past the end) are done
  }

  // the workgroup's waves merged: maxima and sums, then the outputs in four
  // rounds (round r: block rows 4 q + r, W consecutive d per lane)
  float m[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    m[mb] = w.row[mb].max_score(w.lv);
    const float l = sum_quarters(w.row[mb].l) * (1.f / w.vref);
    if (q == 0) {
      lds_m[wave][16 * mb + li] = m[mb];
      lds_l[wave][16 * mb + li] = l;
    }
  }
  __syncthreads();
  if (w.odd) lds_odd = 1;
  // per row: the maximum over the waves, and what the outputs are divided by
  if (tid < ROWS) {
    float mx = lds_m[0][tid], sum = 0.f;
#pragma unroll
    for (int i = 1; i < NW; ++i) mx = fmaxf(mx, lds_m[i][tid]);
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      // (a wave that saw nothing has the sum 0, a row of NaN scores no maximum)
      const float f = lds_m[i][tid] == kNegInf ? 1.f : __builtin_amdgcn_exp2f(lds_m[i][tid] - mx);
      sum += lds_l[i][tid] == 0.f ? 0.f : lds_l[i][tid] * f;
    }
    lds_max[tid] = mx;
    lds_sum[tid] = sum;
  }
  __syncthreads();
  const TreePartials part = tree_partials(a, t, ROWS);
  const int64_t prow0 = ((int64_t)index * t.tiles + tile_row) * ROWS;
  if (!complete && tid < ROWS) {
    float* out = part.ml + (prow0 + tid) * 2;
    out[0] = lds_max[tid];
    out[1] = lds_sum[tid];
  }
  // (an empty range's sums are zero: the merge skips its outputs)
  if (complete || begin < end) {
    float factor[MB];  // this wave's share of its rows
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const int row = 16 * mb + li;
      const float f = m[mb] == kNegInf ? 1.f : __builtin_amdgcn_exp2f(m[mb] - lds_max[row]);
      const float sum = complete ? lds_sum[row] : 1.f;
      factor[mb] = sum == 0.f ? 0.f : f / sum * (1.f / w.vref);
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
          dst[0] = w.acc[mb][c][r] * factor[mb];
          dst[1] = w.acc[mb][c + 1][r] * factor[mb];
        }
      }
      __syncthreads();
      for (int i = tid; i < PAIRS; i += 64 * NW) {
        const int row = i / (2 * W), x = i - row * 2 * W;
        const int qq = x / (W / 2), c = 2 * (x - qq * (W / 2));
        if (row0 + row >= rows) continue;
        float o0 = 0.f, o1 = 0.f;
#pragma unroll
        for (int i4 = 0; i4 < NW; ++i4) {
          o0 += lds_o[i4][row][W * qq + c];
          o1 += lds_o[i4][row][W * qq + c + 1];
        }
        const int d = Tile::v_dim(4 * qq + r, c);  // (c even: d and d + 1)
        const int n = (row0 + row) / group, h = hk * group + (row0 + row - n * group);
        if (FMT != WMX_POOL_INT8 && lds_odd) {
          // drafted values that are not finite, for the queries that see them:
          // any positive weight leaves them as they are
          for (int j = max(begin, range.base); j < end; ++j) {
            if (!tmask[(int64_t)n * a.tree_mask_stride[1] + (j - range.base)] || (kmask && !kmask[j])) continue;
            const char* at = vbase + j * vsb + d * Tile::kElem;
            float v0, v1;
            if constexpr (FMT == WMX_POOL_BF16) {
              v0 = bf16_lo(*(const uint32_t*)at);
              v1 = bf16_hi(*(const uint32_t*)at);
            } else {  // (only NaN)
              const uint32_t u = *(const uint16_t*)at;
              v0 = (u & 0x7fu) == 0x7fu ? __builtin_nanf("") : 0.f;
              v1 = (u & 0x7f00u) == 0x7f00u ? __builtin_nanf("") : 0.f;
            }
            o0 += __builtin_isfinite(v0) ? 0.f : v0;
            o1 += __builtin_isfinite(v1) ? 0.f : v1;
          }
        }
        if (complete) {
          bf16* out = (bf16*)a.o + (int64_t)b * a.o_stride[0] + (int64_t)h * a.o_stride[1] + (int64_t)n * a.o_stride[2] + d;
          *(uint32_t*)out = pack_bf16x2(o0, o1);
        } else {
          float* out = part.o + (prow0 + row) * D + d;
          out[0] = o0;
          out[1] = o1;
        }
      }
    }
  }
}

// Merge of a row's ranges: one thread per four consecutive d, eight ranges'
// loads in flight. `rows_wg`: query rows of a range's workgroup.
__global__ __launch_bounds__(256) void tree_merge_kernel(const wmx_tree_args a, const TreeLaunch t, int rows_wg, int64_t threads) {
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (gid >= threads) return;
  const int D = a.head_dim, per = D / 4, group = a.q_heads / a.kv_heads, rows = a.nodes * group;
  const int64_t row = gid / per;
  const int d = 4 * (int)(gid - row * per);
  const int64_t pair = row / rows;
  const int in_pair = (int)(row - pair * rows), n = in_pair / group;
  const int b = (int)(pair / a.kv_heads), hk = (int)(pair - (int64_t)b * a.kv_heads), h = hk * group + in_pair - n * group;
  const int tile = in_pair / rows_wg;
  int64_t first;
  int count;
  if (t.nsplit > 0) {
    first = pair * t.nsplit;
    count = t.nsplit;
  } else {
    const int* plan = (const int*)a.workspace;
    count = plan[b + 1] - plan[b];
    if (count == 1) return;  // (written by its workgroup)
    first = plan[b] * a.kv_heads + hk * count;
  }
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const TreePartials part = tree_partials(a, t, rows_wg);
  const int64_t part0 = (first * t.tiles + tile) * rows_wg + (in_pair - tile * rows_wg), part_step = (int64_t)t.tiles * rows_wg;
  float mx = kNegInf, sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < count; s0 += 8) {
    f32x2 ml[8];
    f32x4 po[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t r = part0 + min(s0 + u, count - 1) * part_step;
      ml[u] = *(const f32x2*)(part.ml + r * 2);
      po[u] = *(const f32x4*)(part.o + r * D + d);  // an empty range wrote none: not used
    }
    float top = mx;
#pragma unroll
    for (int u = 0; u < 8; ++u) top = fmaxf(top, ml[u][0]);
    const float f = mx == kNegInf ? 1.f : __builtin_amdgcn_exp2f(mx - top);  // (nothing to scale before a first maximum)
    sum *= f;
    o *= f;
    mx = top;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (s0 + u >= count || ml[u][1] == 0.f) continue;
      const float w = ml[u][0] == kNegInf ? 1.f : __builtin_amdgcn_exp2f(ml[u][0] - top);
      sum += ml[u][1] * w;
      o += po[u] * w;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  bf16* out = (bf16*)a.o + (int64_t)b * a.o_stride[0] + (int64_t)h * a.o_stride[1] + (int64_t)n * a.o_stride[2] + d;
  const u32x2 w = {pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
  *(u32x2*)out = w;
}

// Query rows per workgroup: 16 or 32. Two 16s use up to 232 registers, two waves a
// SIMD; three and four share the conversions further but leave one wave a SIMD, and
// took 1.5 and 1.3 times as long (64 nodes x 2 heads over 16 x 8,192 slots).
static int tree_rows(const wmx_tree_args& a) { return (int64_t)a.nodes * (a.q_heads / a.kv_heads) <= 16 ? 16 : 32; }

static TreeLaunch tree_plan(const wmx_tree_args& a) {
  const int64_t rows = (int64_t)a.nodes * (a.q_heads / a.kv_heads), per = tree_rows(a);
  const int64_t tiles = (rows + per - 1) / per, pairs = (int64_t)a.batch * a.kv_heads;
  TreeLaunch t{};
  t.tiles = (int)tiles;
  const bool few = a.capacity <= kOneRange || (a.capacity <= 2 * kOneRange && pairs * tiles >= kCUs);
  t.nsplit = a.num_splits > 0 ? a.num_splits : few || a.batch > kPlanRows || pairs * a.capacity > (1ll << 36) ? 1 : 0;
  t.waves = t.nsplit == 1 && pairs * tiles <= kCUs ? 8 : 4;
  const int64_t step = t.waves * kTreeTile, most = max((int64_t)1, (a.capacity + step - 1) / step);  // steps of a (row, head)
  if (t.nsplit > 0) {
    t.nsplit = (int)min((int64_t)t.nsplit, most);  // (more would be empty)
    t.share = (int)((most + t.nsplit - 1) / t.nsplit);
    t.ranges = (int)min((int64_t)INT32_MAX, pairs * t.nsplit);
  } else {
    const int64_t least = tree_min_share((int)per);
    t.share = (int)max((int64_t)1, tree_dealt((int)per) / tiles);  // workgroups to deal the steps over
    t.ranges = (int)min(pairs + t.share, pairs * ((most + least - 1) / least));
  }
  return t;
}

int64_t tree_workspace_size(const wmx_tree_args& a) {
  const TreeLaunch t = tree_plan(a);
  return t.nsplit == 1 ? 0 : 4 * (kPlanInts + tree_partial_rows(t, tree_rows(a)) * (a.head_dim + 2));
}

template <int FMT, int D, int MB>
static void launch_tree_m(const wmx_tree_args& a, unsigned blocks, const TreeLaunch& t, hipStream_t stream) {
  const dim3 grid(blocks), block(64 * t.waves);
  if (t.waves == 8) hipLaunchKernelGGL((tree_kernel<FMT, D, MB, 8>), grid, block, 0, stream, a, t);
  else hipLaunchKernelGGL((tree_kernel<FMT, D, MB, 4>), grid, block, 0, stream, a, t);
}

template <int FMT, int D>
static void launch_tree_d(const wmx_tree_args& a, unsigned blocks, const TreeLaunch& t, hipStream_t stream) {
  if (tree_rows(a) == 16) launch_tree_m<FMT, D, 1>(a, blocks, t, stream);
  else launch_tree_m<FMT, D, 2>(a, blocks, t, stream);
}

template <int FMT>
static int launch_tree_f(const wmx_tree_args& a, unsigned blocks, const TreeLaunch& t, hipStream_t stream) {
  switch (a.head_dim) {
    case 64: launch_tree_d<FMT, 64>(a, blocks, t, stream); return WMX_OK;
    case 96: launch_tree_d<FMT, 96>(a, blocks, t, stream); return WMX_OK;
    case 128: launch_tree_d<FMT, 128>(a, blocks, t, stream); return WMX_OK;
    default: return WMX_E_UNSUPPORTED;
  }
}

int launch_tree(const wmx_tree_args& a, hipStream_t stream) {
  const TreeLaunch t = tree_plan(a);
  const int64_t blocks = ((int64_t)t.ranges + 7) / 8 * 8 * t.tiles;
  const int64_t merged = (int64_t)a.batch * a.q_heads * a.nodes * (a.head_dim / 4);
  if (blocks > INT32_MAX || (merged + 255) / 256 > INT32_MAX || (int64_t)a.batch * a.kv_heads * max(1, t.nsplit) > INT32_MAX ||
      (int64_t)t.share * max(1, t.nsplit) * t.waves * kTreeTile > INT32_MAX)
    return WMX_E_UNSUPPORTED;  // (ranges are counted, and begin, within 31 bits)
  int rc;
  if (a.format == WMX_POOL_BF16) rc = launch_tree_f<WMX_POOL_BF16>(a, (unsigned)blocks, t, stream);
  else if (a.format == WMX_POOL_E4M3) rc = launch_tree_f<WMX_POOL_E4M3>(a, (unsigned)blocks, t, stream);
  else rc = launch_tree_f<WMX_POOL_INT8>(a, (unsigned)blocks, t, stream);
  if (rc != WMX_OK || t.nsplit == 1) return rc;
  hipLaunchKernelGGL(tree_merge_kernel, dim3((unsigned)((merged + 255) / 256)), dim3(256), 0, stream, a, t, tree_rows(a), merged);
  return WMX_OK;
}

}  // namespace wmx
