// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits, and their gradient (formulas in wmx_attn.h). HBM-bound: the forward
// reads each logit once, the gradient reads it once more and writes it once.
// Measured, 2,048 rows of 151,936 bf16 logits (622 MB): forward 125 us (5.0 TB/s, a
// large read's 6.0) and 5 for the merge, gradient 200 us (6.2 TB/s in and out);
// 37 rows with eight alternatives, a latency, 9.4 and 6.2 us.
//
// Forward: a workgroup takes one chunk of a row, 32 KB that its 256 threads
// hold in registers (eight 16-byte loads each, all in flight at once), so the
// maximum, the sums and the selection pass over registers and not over memory
// again. A chunk leaves (max m, s = sum exp(x - m), t = sum exp(x - m)(x - m))
// and its own top_k, which a second kernel merges per row: with M the largest
// m and S = sum s_c exp(m_c - M), lse = M + log S and
// entropy = log S - sum exp(m_c - M)(t_c + s_c (m_c - M)) / S.
// Everything is fp32; p_j x_j is summed relative to the maximum, so entropies
// of peaked rows do not cancel.
#include "wmx_kernels.h"

namespace wmx {

typedef u32x4 u32x4_any __attribute__((aligned(2)));  // rows of odd vocabularies start anywhere

constexpr int kScoreThreads = 256;
// 16-byte loads per thread and chunk. Forward: 37 rows with alternatives 16 us in
// both kernels, 18 with four loads, 15.3 with sixteen, where the 2,048 rows take
// 130 for 125. Gradient: the 2,048 rows 200 us, 222 with eight; 301 rows of 32,003
// fp32 logits 18.6 us, 23.6 with one.
constexpr int kScoreLoads = 8;
constexpr int kGradLoads = 4;
constexpr int kScoreCandidates = 512;  // room for a chunk's possible top entries
constexpr float kFarBelow = -1.0e4f;    // exp of it is zero; keeps -inf * 0 out of the entropy

template <int DT>
struct Logit {
  static constexpr int kPer = DT == WMX_DTYPE_F32 ? 4 : 8;  // elements of 16 bytes
  static constexpr int kChunk = kScoreThreads * kScoreLoads * kPer;
  static constexpr int kGradChunk = kScoreThreads * kGradLoads * kPer;
  static constexpr int kSize = DT == WMX_DTYPE_F32 ? 4 : 2;

  static __device__ __forceinline__ float one(const void* row, int64_t j) {
    if constexpr (DT == WMX_DTYPE_F32) return ((const float*)row)[j];
    else if constexpr (DT == WMX_DTYPE_BF16) return (float)((const bf16*)row)[j];
    else return (float)((const _Float16*)row)[j];
  }
  static __device__ __forceinline__ void unpack(const u32x4& w, float (&x)[kPer]) {
    if constexpr (DT == WMX_DTYPE_F32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(w[e]);
    } else if constexpr (DT == WMX_DTYPE_BF16) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = bf16_lo(w[e]);
        x[2 * e + 1] = bf16_hi(w[e]);
      }
    } else {
      typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
      const f16x8 h = __builtin_bit_cast(f16x8, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)h[e];
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&x)[kPer]) {
    if constexpr (DT == WMX_DTYPE_F32) {
      return u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
    } else if constexpr (DT == WMX_DTYPE_BF16) {
      return u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
    } else {
      typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
      f16x8 h;
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = (_Float16)x[e];
      return __builtin_bit_cast(u32x4, h);
    }
  }
  static __device__ __forceinline__ void put(void* row, int64_t j, float x) {
    if constexpr (DT == WMX_DTYPE_F32) ((float*)row)[j] = x;
    else if constexpr (DT == WMX_DTYPE_BF16) ((bf16*)row)[j] = (bf16)x;
    else ((_Float16*)row)[j] = (_Float16)x;
  }
  // This thread's N vectors of a chunk, from element j on; all loads in flight at
  // once where the chunk lies whole in the row.
  template <int N>
  static __device__ __forceinline__ void load_chunk(const void* row, int64_t begin, int64_t j, int64_t vocab, u32x4 (&w)[N]) {
    if (begin + kScoreThreads * N * kPer <= vocab) {
      const char* p = (const char*)row + j * kSize;
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = __builtin_nontemporal_load((const u32x4_any*)(p + i * kScoreThreads * 16));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = load(row, j + (int64_t)i * kScoreThreads * kPer, vocab);
    }
  }
  // The vector at element j of a row, -inf past its end.
  static __device__ __forceinline__ u32x4 load(const void* row, int64_t j, int64_t vocab) {
    if (j + kPer <= vocab) {
      return __builtin_nontemporal_load((const u32x4_any*)((const char*)row + j * kSize));
    }
    float x[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = j + e < vocab ? one(row, j + e) : kNegInf;
    return pack(x);
  }
};

// A float's place in the order of the top entries: larger is earlier, NaN
// first, -0 and 0 alike.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  if (x != x) return 0xffffffffu;
  return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
  if (order == 0xffffffffu) return __builtin_nanf("");
  return __uint_as_float((order >> 31) ? order & 0x7fffffffu : ~order);
}
// (value, index) as one key: a larger key is an earlier entry.
__device__ __forceinline__ uint64_t entry_key(float x, int64_t j) {
  return ((uint64_t)order_of(x) << 32) | (uint32_t)~(uint32_t)j;
}
__device__ __forceinline__ int64_t entry_index(uint64_t key) { return (int64_t)(uint32_t)~(uint32_t)key; }

template <class T, class Op>
__device__ __forceinline__ T wave_reduce(T x, Op op) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = op(x, __shfl_xor(x, o));
  return x;
}
template <class T, class Op>
__device__ __forceinline__ T block_reduce(T x, T* lds, Op op) {
  x = wave_reduce(x, op);
  const int w = threadIdx.x >> 6;
  __syncthreads();  // earlier readers of lds are done
  if ((threadIdx.x & 63) == 0) lds[w] = x;
  __syncthreads();
  T r = lds[0];
#pragma unroll
  for (int i = 1; i < kScoreThreads / 64; ++i) r = op(r, lds[i]);
  return r;
}

struct ScorePart {
  float m, s, t, pad;
};

// Writes a row's results from its merged statistics and sorted entries.
__device__ __forceinline__ void finish_row(const wmx_score_args& a, int64_t row, float m, float s, float t, float x_token) {
  const bool empty = m == kNegInf && s == 0.f;
  const float log_s = logf(s);
  const float lse = empty ? kNegInf : m + log_s;
  a.lse[row] = lse;
  a.entropy[row] = empty ? 0.f : log_s - t / s;
  const int64_t token = a.tokens[row];
  float lp;
  if (token == a.ignore_index) lp = 0.f;
  else if (token < 0 || token >= a.vocab) lp = __builtin_nanf("");
  else lp = empty ? kNegInf : (x_token - m) - log_s;
  a.log_probs[row] = lp;
}

template <int DT>
__device__ __forceinline__ float token_logit(const wmx_score_args& a, const void* base, int64_t row) {
  const int64_t token = a.tokens[row];
  return token >= 0 && token < a.vocab ? Logit<DT>::one(base, token) : 0.f;
}

// A chunk's top_k entries in order, by one entry at a time: the largest key
// below the last one. For chunks in which too many values are equal, or too few
// are finite, for the bound below; reads the chunk again for each entry (from
// registers, its keys would take all of them in the common case too).
template <int DT>
__device__ __forceinline__ void select_slowly(const void* base, int64_t j0, int64_t vocab, int k, uint64_t* entries, uint64_t* lds) {
  using L = Logit<DT>;
  constexpr int P = L::kPer;
  uint64_t last = ~0ull;
#pragma unroll 1
  for (int r = 0; r < k; ++r) {
    uint64_t top = 0;
#pragma unroll 1
    for (int i = 0; i < kScoreLoads; ++i) {
      float x[P];
      L::unpack(L::load(base, j0 + (int64_t)i * kScoreThreads * P, vocab), x);
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const int64_t j = j0 + (int64_t)i * kScoreThreads * P + e;
        const uint64_t key = j < vocab ? entry_key(x[e], j) : 0;
        if (key < last && key > top) top = key;
      }
    }
    top = block_reduce(top, lds, [](uint64_t p, uint64_t q) { return p > q ? p : q; });
    if (threadIdx.x == 0) entries[r] = top;  // 0: the chunk has no further entry
    last = top;
  }
}

// Rank of `key` among the first n of `found` (distinct keys), two at a time;
// found[n] exists and is zero where n is odd.
__device__ __forceinline__ int rank_of(uint64_t key, const uint64_t* found, int n) {
  typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
  int rank = 0;
#pragma unroll 4
  for (int i = 0; i < n; i += 2) {
    const u64x2 other = *(const u64x2*)(found + i);
    rank += (other[0] > key) + (other[1] > key);
  }
  return rank;
}

// One chunk of one row. TOP: whether entries are selected.
template <int DT, bool TOP>
__global__ __launch_bounds__(kScoreThreads) void score_kernel(const wmx_score_args a, int chunks) {
  using L = Logit<DT>;
  constexpr int P = L::kPer;
  __shared__ float red[kScoreThreads / 64];
  const int64_t row = blockIdx.x / chunks;
  const int chunk = (int)(blockIdx.x - row * chunks);
  const int tid = threadIdx.x;
  const void* base = (const char*)a.logits + row * a.row_stride * L::kSize;
  const int64_t j0 = (int64_t)chunk * L::kChunk + tid * P;  // this thread's vectors: j0 + i * 256 P

  u32x4 w[kScoreLoads];
  L::load_chunk(base, (int64_t)chunk * L::kChunk, j0, a.vocab, w);

  float best[kScoreLoads], mine = kNegInf;  // of each vector, of all
#pragma unroll
  for (int i = 0; i < kScoreLoads; ++i) {
    float x[P];
    L::unpack(w[i], x);
    best[i] = x[0];
#pragma unroll
    for (int e = 1; e < P; ++e) best[i] = fmaxf(best[i], x[e]);
    mine = fmaxf(mine, best[i]);
  }
  const float m = block_reduce(mine, red, [](float p, float q) { return fmaxf(p, q); });
  const float ref = m == kNegInf ? 0.f : m;
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int i = 0; i < kScoreLoads; ++i) {
    float x[P];
    L::unpack(w[i], x);
#pragma unroll
    for (int e = 0; e < P; ++e) {
      const float d = x[e] - ref;
      const float p = __builtin_amdgcn_exp2f(d * kLog2e);
      s += p;
      t = fmaf(p, fmaxf(d, kFarBelow), t);
    }
  }
  const auto add = [](float p, float q) { return p + q; };
  s = block_reduce(s, red, add);
  t = block_reduce(t, red, add);

  if constexpr (TOP) {
    __shared__ __attribute__((aligned(16))) uint64_t found[kScoreCandidates];
    __shared__ __attribute__((aligned(16))) float quads[64];
    __shared__ uint64_t keys[kScoreThreads / 64];
    __shared__ float bound_lds;
    __shared__ int count;
    const int k = a.top_k;
    uint64_t* entries = (uint64_t*)((ScorePart*)a.workspace + a.rows * chunks) + (row * chunks + chunk) * (int64_t)k;
    // A bound that at least k entries reach: the k-th largest of the maxima of
    // 64 groups of four threads (k <= 32); the entries above it come from
    // fewer than k groups.
    float quad = fmaxf(mine, __shfl_xor(mine, 1));
    quad = fmaxf(quad, __shfl_xor(quad, 2));
    if (tid == 0) count = 0;
    if ((tid & 3) == 0) quads[tid >> 2] = quad;
    __syncthreads();
    if (tid < 64) {
      const float q = quads[tid];
      int above = 0;
#pragma unroll
      for (int i = 0; i < 64; i += 4) {
        const f32x4 o = *(const f32x4*)(quads + i);
#pragma unroll
        for (int u = 0; u < 4; ++u) above += (o[u] > q) + (o[u] == q && i + u < tid);
      }
      if (above == k - 1) bound_lds = q;
    }
    __syncthreads();
    const float bound = bound_lds;
    // (a chunk with a NaN or +inf has the sum NaN)
    const bool plain = bound > kNegInf && s == s;
    if (plain && mine >= bound) {
#pragma unroll
      for (int i = 0; i < kScoreLoads; ++i) {
        if (best[i] < bound) continue;
        float x[P];
        L::unpack(w[i], x);
#pragma unroll
        for (int e = 0; e < P; ++e) {
          if (x[e] < bound) continue;  // (past the row's end: -inf)
          const int at = atomicAdd(&count, 1);
          if (at < kScoreCandidates) found[at] = entry_key(x[e], j0 + (int64_t)i * kScoreThreads * P + e);
        }
      }
    }
    __syncthreads();
    const int n = count;
    if (plain && n <= kScoreCandidates) {
      if (tid == 0 && (n & 1)) found[n] = 0;  // (n odd is below the capacity, which is even)
      __syncthreads();
      for (int c = tid; c < n; c += kScoreThreads) {
        const uint64_t key = found[c];
        const int rank = rank_of(key, found, n);
        if (rank < k) entries[rank] = key;
      }
    } else {
      select_slowly<DT>(base, j0, a.vocab, k, entries, keys);
    }
  }
  if (tid == 0) {
    if (chunks > 1 || TOP) ((ScorePart*)a.workspace)[row * chunks + chunk] = ScorePart{m, s, t, 0.f};
    else finish_row(a, row, m, s, t, token_logit<DT>(a, base, row));
  }
}

// One wave per row: the chunks' statistics and sorted entries merged.
constexpr int kMergeEntries = 1024;  // entries of a row that are merged in LDS
template <int DT>
__global__ __launch_bounds__(64) void score_merge_kernel(const wmx_score_args a, int chunks) {
  __shared__ __attribute__((aligned(16))) uint64_t found[kMergeEntries + 2];
  __shared__ int count;
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x, k = a.top_k;
  const int64_t n = (int64_t)chunks * k;
  const ScorePart* parts = (const ScorePart*)a.workspace + row * chunks;
  const uint64_t* entries = (const uint64_t*)((const ScorePart*)a.workspace + a.rows * chunks) + row * n;
  const void* base = (const char*)a.logits + row * a.row_stride * Logit<DT>::kSize;
  const float x_token = token_logit<DT>(a, base, row);
  const auto largest = [](auto p, auto q) { return p > q ? p : q; };
  float m = kNegInf;
  for (int c = lane; c < chunks; c += 64) m = fmaxf(m, parts[c].m);
  // A bound that at least k entries reach, and its entries: each chunk has
  // ceil(k / chunks) of them at or above the least of the chunks' such entries.
  const bool in_lds = k > 0 && n <= kMergeEntries;
  if (in_lds) {
    const int each = (k + chunks - 1) / chunks;
    uint64_t least = ~0ull;
    for (int c = lane; c < chunks; c += 64) {
      const uint64_t e = entries[(int64_t)c * k + each - 1];
      least = e < least ? e : least;
    }
    least = ~wave_reduce(~least, largest);
    if (lane == 0) count = 0;
    __syncthreads();
    for (int i = lane; i < n; i += 64) {
      const uint64_t e = entries[i];
      if (e >= least && e != 0) found[atomicAdd(&count, 1)] = e;
    }
  }
  m = wave_reduce(m, [](float p, float q) { return fmaxf(p, q); });
  const float ref = m == kNegInf ? 0.f : m;
  float s = 0.f, t = 0.f;
  for (int c = lane; c < chunks; c += 64) {
    const float d = parts[c].m - ref;
    const float f = __builtin_amdgcn_exp2f(d * kLog2e);
    s += parts[c].s * f;
    t += f * (parts[c].t + parts[c].s * fmaxf(d, kFarBelow));
  }
  const auto add = [](float p, float q) { return p + q; };
  s = wave_reduce(s, add);
  t = wave_reduce(t, add);
  if (lane == 0) finish_row(a, row, m, s, t, x_token);
  if (k == 0) return;
  const float log_s = logf(s);
  const bool empty = m == kNegInf && s == 0.f;
  const auto put = [&](int rank, uint64_t key) {
    a.top_indices[row * k + rank] = entry_index(key);
    a.top_log_probs[row * k + rank] = empty ? kNegInf : (value_of((uint32_t)(key >> 32)) - ref) - log_s;
  };
  if (in_lds) {
    __syncthreads();
    const int found_n = count;
    if (lane == 0) found[found_n] = 0;
    __syncthreads();
    for (int c = lane; c < found_n; c += 64) {
      const uint64_t key = found[c];
      const int rank = rank_of(key, found, found_n);
      if (rank < k) put(rank, key);
    }
    return;
  }
  // rows of very many chunks: the next of all entries k times, the largest key
  // below the last
  uint64_t last = ~0ull;
  for (int r = 0; r < k; ++r) {
    uint64_t top = 0;
    for (int64_t i = lane; i < n; i += 64) {
      const uint64_t key = entries[i];
      if (key < last && key > top) top = key;
    }
    top = wave_reduce(top, largest);
    if (lane == 0) put(r, top);
    last = top;
  }
}

// The gradient: p (slope) for every logit of a chunk, then the chunk's few
// named positions once more with what reaches their log probabilities.
template <int DT>
__global__ __launch_bounds__(kScoreThreads) void score_bwd_kernel(const wmx_score_args a, int chunks) {
  using L = Logit<DT>;
  constexpr int P = L::kPer;
  const int64_t row = blockIdx.x / chunks;
  const int chunk = (int)(blockIdx.x - row * chunks);
  const int tid = threadIdx.x, k = a.top_k;
  const void* base = (const char*)a.logits + row * a.row_stride * L::kSize;
  void* out = (char*)a.grad_logits + row * (int64_t)a.vocab * L::kSize;
  const int64_t begin = (int64_t)chunk * L::kGradChunk, j0 = begin + tid * P;

  u32x4 w[kGradLoads];
  L::load_chunk(base, begin, j0, a.vocab, w);

  const float lse = a.lse[row], entropy = a.entropy[row];
  const int64_t token = a.tokens[row];
  float g_token = a.grad_log_probs && token != a.ignore_index ? a.grad_log_probs[row] : 0.f;
  if (token != a.ignore_index && (token < 0 || token >= a.vocab) && a.grad_log_probs) g_token = __builtin_nanf("");
  const float g_entropy = a.grad_entropy ? a.grad_entropy[row] : 0.f;
  float sum = g_token;
  if (a.grad_top)
    for (int i = 0; i < k; ++i) sum += a.grad_top[row * k + i];
  const bool empty = lse == kNegInf;
  const auto slope = [&](float x) {
    const float d = x - lse;
    const float p = __builtin_amdgcn_exp2f(d * kLog2e);
    const float g = -p * fmaf(g_entropy, d + entropy, sum);
    return empty || p == 0.f ? 0.f : g;
  };
#pragma unroll
  for (int i = 0; i < kGradLoads; ++i) {
    const int64_t j = j0 + (int64_t)i * kScoreThreads * P;
    if (j >= a.vocab) break;
    float x[P];
    L::unpack(w[i], x);
#pragma unroll
    for (int e = 0; e < P; ++e) x[e] = slope(x[e]);
    if (j + P <= a.vocab) {
      __builtin_nontemporal_store(L::pack(x), (u32x4_any*)((char*)out + j * L::kSize));
    } else {
#pragma unroll
      for (int e = 0; e < P; ++e)
        if (j + e < a.vocab) L::put(out, j + e, x[e]);
    }
  }
  __builtin_amdgcn_s_waitcnt(0);  // the stores above have landed: the ones below replace some
  __syncthreads();
  if (tid > k || empty) return;
  const int64_t at = tid == k ? (a.grad_log_probs && token != a.ignore_index ? token : -1)
                              : (a.grad_top ? a.top_indices[row * k + tid] : -1);
  if (at < begin || at >= begin + L::kGradChunk || at >= a.vocab) return;
  float g = slope(L::one(base, at));
  if (at == token) g += g_token;
  if (a.grad_top)
    for (int i = 0; i < k; ++i)
      if (a.top_indices[row * k + i] == at) g += a.grad_top[row * k + i];
  L::put(out, at, g);
}

template <int DT>
int64_t score_chunks_of(const wmx_score_args& a) {
  return ((int64_t)a.vocab + Logit<DT>::kChunk - 1) / Logit<DT>::kChunk;
}
static int64_t score_chunks(const wmx_score_args& a) {
  return a.dtype == WMX_DTYPE_F32 ? score_chunks_of<WMX_DTYPE_F32>(a) : score_chunks_of<WMX_DTYPE_BF16>(a);
}

int64_t score_workspace_size(const wmx_score_args& a) {
  return a.rows * score_chunks(a) * (int64_t)(sizeof(ScorePart) + a.top_k * sizeof(uint64_t));
}

template <int DT>
static int launch_score_t(const wmx_score_args& a, hipStream_t stream) {
  const int64_t chunks = score_chunks(a);
  if (a.rows * chunks > INT32_MAX) return WMX_E_UNSUPPORTED;
  const dim3 grid((unsigned)(a.rows * chunks));
  if (a.top_k)
    hipLaunchKernelGGL((score_kernel<DT, true>), grid, dim3(kScoreThreads), 0, stream, a, (int)chunks);
  else
    hipLaunchKernelGGL((score_kernel<DT, false>), grid, dim3(kScoreThreads), 0, stream, a, (int)chunks);
  if (chunks > 1 || a.top_k)
    hipLaunchKernelGGL((score_merge_kernel<DT>), dim3((unsigned)a.rows), dim3(64), 0, stream, a, (int)chunks);
  return WMX_OK;
}

int launch_score(const wmx_score_args& a, hipStream_t stream) {
  if (a.dtype == WMX_DTYPE_F32) return launch_score_t<WMX_DTYPE_F32>(a, stream);
  if (a.dtype == WMX_DTYPE_BF16) return launch_score_t<WMX_DTYPE_BF16>(a, stream);
  return launch_score_t<WMX_DTYPE_F16>(a, stream);
}

template <int DT>
static int launch_score_bwd_t(const wmx_score_args& a, hipStream_t stream) {
  const int64_t chunks = ((int64_t)a.vocab + Logit<DT>::kGradChunk - 1) / Logit<DT>::kGradChunk;
  if (a.rows * chunks > INT32_MAX) return WMX_E_UNSUPPORTED;
  hipLaunchKernelGGL((score_bwd_kernel<DT>), dim3((unsigned)(a.rows * chunks)), dim3(kScoreThreads), 0, stream, a, (int)chunks);
  return WMX_OK;
}

int launch_score_bwd(const wmx_score_args& a, hipStream_t stream) {
  if (a.dtype == WMX_DTYPE_F32) return launch_score_bwd_t<WMX_DTYPE_F32>(a, stream);
  if (a.dtype == WMX_DTYPE_BF16) return launch_score_bwd_t<WMX_DTYPE_BF16>(a, stream);
  return launch_score_bwd_t<WMX_DTYPE_F16>(a, stream);
}

}  // namespace wmx
