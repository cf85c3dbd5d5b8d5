// Low-rank adapters of many requests beside one shared projection:
//   y[t] = x[t] W^T + scale_a (x[t] A_a^T) B_a^T,   a = index[t]  (outside of the bank: x[t] W^T)
// with A [slots, rank, K] and B [slots, N, rank] as stored.
//
// What it has to read beside the projection is small (a rank of 16 beside 4,096 -> 4,096: 1/128 of W for
// every adapter in the step), so what counts is that the projection's kernels run as they do without it.
//   Where the projection itself runs as the paired tcgen05 product (hundreds of tokens, bfloat16):
//   `adapter_low` (adapter_tcgen05.cu) makes the rank numbers of each block of 256 tokens as planes, one for
//   every adapter that has tokens in the block (zero in the rows of others), and the product takes them as
//   more K behind its own, [x | planes] [W | B]^T: one sum in tensor memory, one rounding
//   (gemm_tcgen05_pair.cu, MoreK). A rank number goes there as the sum of two bfloat16 numbers
//   (adapter_planes.cuh), 16 bits of it, and its rounding is 2^-16 of the adapter's part at most, a 256th of a
//   bfloat16 result's own. (Rounded to one bfloat16 number: 16.8 us where 18.6 stands below, 2,048 tokens the same.)
//   Up to 64 tokens, bfloat16, few adapters (below 17 only beside wide projections): the same with planes by
//   `adapter_shrink` behind the K of the product that shares K in a cluster (gemm_rows_tcgen05.cu, RowsMore):
//   48 tokens of 4,096 -> 4,096 with 12 adapters of rank 64 18.6 us, 19.6 with a pass of its own for the sums;
//   10.1 without adapters.
//   Else up to 16 tokens, bfloat16: `adapter_shrink` leaves them as 32-bit rows, and the weight-streaming product
//   adds their product with B to its sums in front of its epilogue (gemm_skinny.cu, ADAPT). Nothing is rounded in
//   between.
//   Else: `adapter_shrink` (or, for many numbers, `adapter_low`) leaves them as 32-bit rows, the projection
//   leaves 32-bit sums (split-K planes), and `adapter_expand` adds up sums and adapters and rounds once.
#include "adapter_planes.cuh"
#include "common.cuh"

namespace {

constexpr int THREADS = 256;

__device__ __forceinline__ uint4 ld16(const void* p) {  // never by the non-coherent path
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ float dot8(const uint4& a, const uint4& b, float sum) {  // eight bfloat16 pairs
  const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&a);
  const __nv_bfloat162* y = reinterpret_cast<const __nv_bfloat162*>(&b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = __bfloat1622float2(x[i]), v = __bfloat1622float2(y[i]);
    sum = fmaf(u.x, v.x, sum);
    sum = fmaf(u.y, v.y, sum);
  }
  return sum;
}

// The rank numbers as planes for a product that takes them as more K (fb_gemm_rows_adapted): adapter by
// adapter [256 rows, fb_plane_width(rank)] bfloat16, zero in the rows of other adapters' tokens.
struct ShrinkPlanes {
  __nv_bfloat16* u;
  int* counts;    // [1]: adapters with tokens
  int* slots_of;  // which they are, in ascending order
};
constexpr int PLANE_ROWS = 256, PLANE_SLOTS = 1024;

// low[t, j] = scale * sum_k x[t, k] A[a][j, k]. A warp has four ranks, so that a piece of x in its registers meets
// four rows of A, and PARTS warps of a block share K; block (i, t) has the ranks from i * BLOCK_RANKS on. Few
// numbers take many warps each, for a warp's loads are then two rounds, all under way together; many have
// enough warps without. The whole operator (planes of one number a rank) with 8, 4, 2 and 1 parts: 8 tokens of
// 14,336, rank 64, 27.6, 31, 34 and 46 us; 48 of 4,096, rank 64, 17.6, 16.9, 18.9 and 22.4; 128 of 2,048, rank 64, 24.8, 21.0, 20.5 and 20.6. (A rank
// a warp: 33, 17.1 and 19.6, and 64 tokens of 14,336 82 us against 47.) `wide`: rows are on 16-byte boundaries.
// PLANES: the numbers go to the token's row of its adapter's plane, and zeros to its row of the others.
constexpr int RANKS = 4;  // of a warp
template <typename T, int PARTS, bool PLANES>
__global__ void __launch_bounds__(THREADS)
adapter_shrink_kernel(const T* x, long long ldx, const T* a, const float* scales, const int* index, int slots,
                      int rank, int K, int wide, float* low, const ShrinkPlanes planes) {
  constexpr int WARPS = THREADS / 32;
  constexpr int BLOCK_RANKS = RANKS * WARPS / PARTS;
  __shared__ float sums[BLOCK_RANKS][PARTS];
  fb_pdl_wait();
  fb_pdl_launch();
  const int t = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, j0 = blockIdx.x * BLOCK_RANKS;
  const int share = warp % PARTS, first = warp / PARTS * RANKS;  // of the block's ranks
  const int slot = index[t];
  const bool own = slot >= 0 && slot < slots;
  __shared__ int s_order;
  if constexpr (PLANES) {
    __shared__ unsigned s_present[PLANE_SLOTS / 32];
    __shared__ int s_count;
    const int tid = threadIdx.x;
    if (tid < PLANE_SLOTS / 32) s_present[tid] = 0u;
    __syncthreads();
    if (tid < (int)gridDim.y) {  // (256 tokens at most)
      const int other = index[tid];
      if (other >= 0 && other < slots) atomicOr(&s_present[other >> 5], 1u << (other & 31));
    }
    __syncthreads();
    if (warp == 0) {
      const unsigned marks = s_present[lane];
      const int here = __popc(marks), word = own ? slot >> 5 : 0;
      const unsigned below = own ? (1u << (slot & 31)) - 1 : 0u;
      const int count = __reduce_add_sync(0xffffffffu, here);
      const int order = __reduce_add_sync(0xffffffffu, lane < word ? here : lane == word ? __popc(marks & below) : 0);
      if (lane == 0) {
        s_count = count;
        s_order = order;
      }
      if (blockIdx.x == 0 && t == 0) {
        int at = here;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int front = __shfl_up_sync(0xffffffffu, at, o);
          if (lane >= o) at += front;
        }
        at -= here;
        for (unsigned left = marks; left != 0u; left &= left - 1) planes.slots_of[at++] = lane * 32 + __ffs(left) - 1;
        if (lane == 0) planes.counts[0] = count;
      }
    }
    __syncthreads();
    // (the last block's part reaches to the end of the last 32 ranks)
    const int live = (j0 + BLOCK_RANKS >= rank ? fb_plane_ranks(rank) : j0 + BLOCK_RANKS) - j0;
    for (int i = tid; i < s_count * live; i += THREADS) {
      const int e = i / live, j = j0 + i % live;
      if (!own || e != s_order || j >= rank)
        fb_store_halves(planes.u + ((size_t)e * PLANE_ROWS + t) * fb_plane_width(rank), j, 0.f);
    }
  }
  if (!own) return;  // (the whole block)
  constexpr int EACH = 16 / sizeof(T), ROUND = 32 * EACH;
  const int rounds = (K + ROUND - 1) / ROUND, each = (rounds + PARTS - 1) / PARTS;
  const int from = share * each * ROUND, to = min(K, from + each * ROUND);
  const T* row = x + (size_t)t * ldx;
  const T* w[RANKS];
#pragma unroll
  for (int q = 0; q < RANKS; ++q) w[q] = a + ((size_t)slot * rank + min(j0 + first + q, rank - 1)) * K;
  float sum[RANKS] = {};
  int k = from + lane * EACH;
  if (wide) {
    constexpr int AHEAD = 2;
    for (; k < to; k += AHEAD * ROUND) {  // (K is a multiple of EACH)
      uint4 u[AHEAD], v[AHEAD][RANKS];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const bool in = k + i * ROUND < to;
        u[i] = in ? ld16(row + k + i * ROUND) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int q = 0; q < RANKS; ++q) v[i][q] = in ? ld16(w[q] + k + i * ROUND) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
#pragma unroll
        for (int q = 0; q < RANKS; ++q) {
          if constexpr (sizeof(T) == 2) {
            sum[q] = dot8(u[i], v[i][q], sum[q]);
          } else {
            const float* f = reinterpret_cast<const float*>(&u[i]);
            const float* g = reinterpret_cast<const float*>(&v[i][q]);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[q] = fmaf(f[e], g[e], sum[q]);
          }
        }
      }
    }
  } else {
    for (; k < to; k += ROUND) {
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        if (k + e >= to) break;
        const float f = fb_load_coherent(row + k + e);
#pragma unroll
        for (int q = 0; q < RANKS; ++q) sum[q] = fmaf(f, fb_load_coherent(w[q] + k + e), sum[q]);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < RANKS; ++q) {
    sum[q] = fb_warp_sum(sum[q]);
    if (lane == 0) sums[first + q][share] = sum[q];
  }
  __syncthreads();
  if (threadIdx.x < BLOCK_RANKS && j0 + (int)threadIdx.x < rank) {
    const int j = j0 + threadIdx.x;
    float whole = 0.f;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) whole += sums[threadIdx.x][i];
    whole *= scales[slot];
    if constexpr (PLANES) fb_store_halves(planes.u + ((size_t)s_order * PLANE_ROWS + t) * fb_plane_width(rank), j, whole);
    else low[(size_t)t * rank + j] = whole;
  }
}

template <typename T, bool PLANES>
void launch_shrink(const T* x, long long ldx, const T* a, const float* scales, const int* index, int slots,
                   int rank, int tokens, int K, int wide, float* low, const ShrinkPlanes& planes, cudaStream_t stream) {
  auto launch = [&](auto kernel, int ranks) {
    fb_launch(kernel, dim3((rank + ranks - 1) / ranks, tokens), dim3(THREADS), 0, stream, x, ldx, a, scales, index,
              slots, rank, K, wide, low, planes);
  };
  constexpr int ALL = RANKS * THREADS / 32;
  const long long numbers = (long long)tokens * rank;
  if (numbers <= 1024) launch(adapter_shrink_kernel<T, 8, PLANES>, ALL / 8);
  else if (numbers <= 4096) launch(adapter_shrink_kernel<T, 4, PLANES>, ALL / 4);
  else launch(adapter_shrink_kernel<T, 2, PLANES>, ALL / 2);
}

// out[t, n] = sum over the planes of base[., t, n] + sum_j low[t, j] B[a][n, j].
//
// A row of B is read by L neighbouring lanes, 16 bytes each, so that a load of the warp takes 512 bytes that
// lie side by side (a thread a feature, which reads its row alone, made 32 lines of every load: 48 tokens,
// 4,096 features, rank 64, 11 us for the kernel). A lane keeps its few ranks' numbers of a token, multiplies
// L features, and the lanes exchange sums so that each ends with the whole sum of one feature.
constexpr int EXPAND_THREADS = 128;
template <int L> constexpr int ROUNDS_OF = L >= 4 ? 1 : 4 / L;  // of 32 features a warp

template <typename T>
__device__ __forceinline__ void unpack(const uint4& q, float (&f)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 2) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 v = __bfloat1622float2(h[e]);
      f[2 * e] = v.x;
      f[2 * e + 1] = v.y;
    }
  } else {
    const float4 v = *reinterpret_cast<const float4*>(&q);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  }
}

// L sums a lane, one a feature -> the sum over the L lanes of the lane's own feature.
template <int L>
__device__ __forceinline__ float share_out(float (&v)[L], int li) {
#pragma unroll
  for (int s = L / 2; s > 0; s >>= 1) {
    const bool upper = (li & s) != 0;
#pragma unroll
    for (int i = 0; i < s; ++i) {
      const float send = upper ? v[i] : v[i + s], keep = upper ? v[i + s] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, s);
    }
  }
  return v[0];
}

template <typename T, typename Out, int L, int TOKENS>
__global__ void __launch_bounds__(EXPAND_THREADS, L <= 8 ? 6 : 3)
adapter_expand_kernel(const float* base, int planes, long long plane_stride, long long ldb, const float* low,
                      const T* b, const int* index, int slots, int rank, int tokens, int N, Out* out,
                      long long ldo) {
  constexpr int EACH = 16 / sizeof(T), ROUNDS = ROUNDS_OF<L>, GROUPS = 32 / L;
  extern __shared__ __align__(16) float mine[];  // [TOKENS][rank]
  __shared__ int s_slot[TOKENS];
  fb_pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, li = lane % L, group = lane / L;
  const int t0 = blockIdx.y * TOKENS, live = min(TOKENS, tokens - t0);
  const int n0 = (blockIdx.x * (EXPAND_THREADS / 32) + (tid >> 5)) * 32 * ROUNDS;
  if (tid < TOKENS) {
    const int slot = tid < live ? index[t0 + tid] : -1;
    s_slot[tid] = slot < slots ? slot : -1;
  }
  // what the projection left for this lane's features
  float sum[TOKENS][ROUNDS];
#pragma unroll
  for (int t = 0; t < TOKENS; ++t)
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const int n = n0 + r * 32 + li * GROUPS + group;
      sum[t][r] = t < live && n < N ? __ldcg(base + (size_t)(t0 + t) * ldb + n) : 0.f;
    }
  for (int i = tid; i < live * rank / 4; i += EXPAND_THREADS)  // (rows of tokens without an adapter go unused)
    reinterpret_cast<float4*>(mine)[i] = __ldcg(reinterpret_cast<const float4*>(low + (size_t)t0 * rank) + i);
#pragma unroll 2
  for (int p = 1; p < planes; ++p)
#pragma unroll
    for (int t = 0; t < TOKENS; ++t)
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) {
        const int n = n0 + r * 32 + li * GROUPS + group;
        if (t < live && n < N) sum[t][r] += __ldcg(base + (size_t)p * plane_stride + (size_t)(t0 + t) * ldb + n);
      }
  __syncthreads();
  auto row_at = [&](int slot, int r, int i) {  // (features past the last one read the last one's row)
    return b + ((size_t)slot * N + min(n0 + r * 32 + i * GROUPS + group, N - 1)) * rank;
  };
  if constexpr (L <= 8) {  // four or eight rows a lane, kept from token to token as they are stored
    uint4 raw[ROUNDS * L];
    int there = -1;
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) {
      const int slot = s_slot[t];
      if (slot < 0) continue;
      const bool in = li * EACH < rank;
      if (slot != there) {
#pragma unroll
        for (int i = 0; i < ROUNDS * L; ++i)
          raw[i] = in ? ld16(row_at(slot, i / L, i % L) + li * EACH) : make_uint4(0u, 0u, 0u, 0u);
        there = slot;
      }
      float f[EACH];
#pragma unroll
      for (int e = 0; e < EACH; ++e) f[e] = in ? mine[t * rank + li * EACH + e] : 0.f;
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) {
        float v[L];
#pragma unroll
        for (int i = 0; i < L; ++i) {
          float w[EACH];
          unpack<T>(raw[r * L + i], w);
          v[i] = w[0] * f[0];
#pragma unroll
          for (int e = 1; e < EACH; ++e) v[i] = fmaf(w[e], f[e], v[i]);
        }
        sum[t][r] += share_out<L>(v, li);
      }
    }
  } else {
    for (int t = 0; t < live; ++t) {
      const int slot = s_slot[t];
      if (slot < 0) continue;
      float v[L];
#pragma unroll
      for (int i = 0; i < L; ++i) v[i] = 0.f;
      for (int j = li * EACH; j - li * EACH < rank; j += L * EACH) {
        const bool in = j < rank;
        float f[EACH];
#pragma unroll
        for (int e = 0; e < EACH; ++e) f[e] = in ? mine[t * rank + j + e] : 0.f;
#pragma unroll
        for (int i0 = 0; i0 < L; i0 += 8) {
          uint4 raw[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) raw[i] = in ? ld16(row_at(slot, 0, i0 + i) + j) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float w[EACH];
            unpack<T>(raw[i], w);
#pragma unroll
            for (int e = 0; e < EACH; ++e) v[i0 + i] = fmaf(w[e], f[e], v[i0 + i]);
          }
        }
      }
      const float whole = share_out<L>(v, li);
#pragma unroll
      for (int q = 0; q < TOKENS; ++q)  // (registers have no runtime index)
        if (q == t) sum[q][0] += whole;
    }
  }
#pragma unroll
  for (int t = 0; t < TOKENS; ++t)
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const int n = n0 + r * 32 + li * GROUPS + group;
      if (t < live && n < N) out[(size_t)(t0 + t) * ldo + n] = fb_from_float<Out>(sum[t][r]);
    }
}

// Tokens a block: one until that makes more blocks than the SMs hold at a time, then two or four, which
// reuse a row of B where neighbours share it (2,048 -> 4,096, rank 16, 4 adapters, the whole operator with one,
// two and four: 17 tokens 11.0, 11.4, 11.6 us; 128 tokens 15.8, 14.5, 15.1; 256 21.2, 19.1, 18.0; 2,048 ->
// 28,672, rank 32, 64 tokens 48, 42, 40. With eight: 15.3 at 64 tokens against 13.3, and never ahead by 2%).
template <typename T, typename Out, int L>
void launch_expand(const float* base, int planes, long long plane_stride, long long ldb, const float* low,
                   const T* b, const int* index, int slots, int rank, int tokens, int N, Out* out, long long ldo,
                   cudaStream_t stream) {
  constexpr int FEATURES = EXPAND_THREADS * ROUNDS_OF<L>;
  const int columns = (N + FEATURES - 1) / FEATURES;
  const long long once = 12LL * sm_count();
  auto launch = [&](auto kernel, int each) {
    fb_launch(kernel, dim3(columns, (tokens + each - 1) / each), dim3(EXPAND_THREADS), (size_t)each * rank * 4,
              stream, base, planes, plane_stride, ldb, low, b, index, slots, rank, tokens, N, out, ldo);
  };
  if ((long long)columns * tokens <= once) launch(adapter_expand_kernel<T, Out, L, 1>, 1);
  else if ((long long)columns * tokens <= 2 * once) launch(adapter_expand_kernel<T, Out, L, 2>, 2);
  else launch(adapter_expand_kernel<T, Out, L, 4>, 4);
}

// As many lanes a row of B as it has pieces of 16 bytes (a power of two, 32 at most).
template <typename T, typename Out>
void expand_by_rank(const float* base, int planes, long long plane_stride, long long ldb, const float* low,
                    const T* b, const int* index, int slots, int rank, int tokens, int N, Out* out,
                    long long ldo, cudaStream_t stream) {
  const int pieces = rank / (16 / (int)sizeof(T));
#define FB_EXPAND(L) \
  launch_expand<T, Out, L>(base, planes, plane_stride, ldb, low, b, index, slots, rank, tokens, N, out, ldo, stream)
  if (pieces <= 1) FB_EXPAND(1);
  else if (pieces <= 2) FB_EXPAND(2);
  else if (pieces <= 4) FB_EXPAND(4);
  else if (pieces <= 8) FB_EXPAND(8);
  else if (pieces <= 16) FB_EXPAND(16);
  else FB_EXPAND(32);
#undef FB_EXPAND
}
}  // namespace

FB_API int fb_adapter_shrink(const void* x, long long ldx, int dtype, const void* a, const float* scales,
                             const int* index, int slots, int rank, int T, int K, float* low,
                             cudaStream_t stream) {
  FB_REQUIRE(T >= 0 && T <= 65535 && K > 0 && rank > 0 && slots > 0 && ldx >= K,
             "adapter_shrink: bad sizes T=%d K=%d rank=%d", T, K, rank);
  if (T == 0) return 0;
  const int each = dtype == FB_BF16 ? 8 : 4;
  const int wide = K % each == 0 && ldx % each == 0 && (((uintptr_t)x | (uintptr_t)a) % 16) == 0;
  FB_DISPATCH_DTYPE(dtype, E, launch_shrink<E, false>((const E*)x, ldx, (const E*)a, scales, index, slots, rank, T, K,
                                                      wide, low, ShrinkPlanes{}, stream));
  return fb_check_launch("adapter_shrink");
}

// The same as planes: u [adapters with tokens * 256, fb_plane_width(rank)], counts [1], slots_of [the same number].
// Up to 256 tokens, bfloat16; rows behind the last token are left as they are.
FB_API int fb_adapter_shrink_planes(const void* x, long long ldx, const void* a, const float* scales,
                                    const int* index, int slots, int rank, int T, int K, void* u, int* counts,
                                    int* slots_of, cudaStream_t stream) {
  FB_REQUIRE(T > 0 && T <= PLANE_ROWS && K > 0 && rank > 0 && slots > 0 && slots <= PLANE_SLOTS && ldx >= K,
             "adapter_shrink_planes: bad sizes T=%d K=%d rank=%d slots=%d", T, K, rank, slots);
  const int wide = K % 8 == 0 && ldx % 8 == 0 && (((uintptr_t)x | (uintptr_t)a) % 16) == 0;
  launch_shrink<__nv_bfloat16, true>((const __nv_bfloat16*)x, ldx, (const __nv_bfloat16*)a, scales, index, slots,
                                     rank, T, K, wide, nullptr, ShrinkPlanes{(__nv_bfloat16*)u, counts, slots_of},
                                     stream);
  return fb_check_launch("adapter_shrink_planes");
}

FB_API int fb_adapter_expand(const float* base, int planes, long long plane_stride, long long ldb,
                             const float* low, const void* b, int dtype, const int* index, int slots, int rank,
                             int T, int N, void* out, int out_dtype, long long ldo, cudaStream_t stream) {
  FB_REQUIRE(T >= 0 && N > 0 && rank > 0 && rank <= 512 && rank % 8 == 0 && slots > 0 && planes > 0 && ldb >= N &&
                 ldo >= N && (((uintptr_t)b | (uintptr_t)low) % 16) == 0,
             "adapter_expand: bad sizes T=%d N=%d rank=%d, or operands not on 16-byte boundaries", T, N, rank);
  FB_REQUIRE(T <= 65535, "adapter_expand: %d tokens (65535 at most)", T);
  if (T == 0) return 0;
  FB_DISPATCH_DTYPE(dtype, E, FB_DISPATCH_DTYPE(out_dtype, O,
      expand_by_rank(base, planes, plane_stride, ldb, low, (const E*)b, index, slots, rank, T, N, (O*)out, ldo,
                     stream)));
  return fb_check_launch("adapter_expand");
}
