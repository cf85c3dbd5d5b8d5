// Low-rank adapters of many requests beside one shared projection:
//   y[t] = x[t] W^T + scale_a (x[t] A_a^T) B_a^T,   a = index[t]  (outside of the bank: x[t] W^T)
// with A [slots, rank, K] and B [slots, N, rank] as stored.
//
// What it has to read beside the projection is small (a rank of 16 beside 4,096 -> 4,096: 1/128 of W for
// every adapter in the step), so what counts is that the projection's kernels run as they do without it.
//   Where the projection itself runs as the paired tcgen05 product (hundreds of tokens, bfloat16):
//   `adapter_low` (adapter_tcgen05.cu) makes the rank numbers of each block of 256 tokens as planes, one for every adapter that
//   has tokens in the block (zero in the rows of others), and the product takes them as more K behind its
//   own, [x | planes] [W | B]^T: one sum in tensor memory, one rounding (gemm_tcgen05_pair.cu, MoreK). The
//   rank numbers are rounded to bfloat16 for that, 2^-9 of the adapter's part on average.
//   More than 16 tokens, else: `adapter_low` leaves them as 32-bit rows, the projection leaves 32-bit sums
//   (split-K planes), and `adapter_expand_mma` adds up sums and adapters on the tensor cores (again of
//   bfloat16 rank numbers) and rounds once.
//   A few tokens, and float32: the same in three with plain multiply-adds, nothing rounded in between.
#include "common.cuh"

namespace {

constexpr int THREADS = 256;

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
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

// Block (j, t): low[t, 8 j + warp] = scale * sum_k x[t, k] A[a][.., k], a warp a rank. `wide`: rows are
// on 16-byte boundaries.
template <typename T>
__global__ void __launch_bounds__(THREADS)
adapter_shrink_kernel(const T* x, long long ldx, const T* a, const float* scales, const int* index, int slots,
                      int rank, int K, int wide, float* low) {
  fb_pdl_wait();
  fb_pdl_launch();
  const int t = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j = blockIdx.x * (THREADS / 32) + warp;
  const int slot = index[t];
  if (slot < 0 || slot >= slots || j >= rank) return;
  const T* row = x + (size_t)t * ldx;
  const T* w = a + ((size_t)slot * rank + j) * K;
  constexpr int EACH = 16 / sizeof(T);
  float sum = 0.f;
  int k = lane * EACH;
  if (wide) {
    constexpr int AHEAD = 4;
    for (; k + (AHEAD - 1) * 32 * EACH < K; k += AHEAD * 32 * EACH) {  // (K is a multiple of EACH)
      uint4 u[AHEAD], v[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        v[i] = ld16(w + k + i * 32 * EACH);
        u[i] = ld16(row + k + i * 32 * EACH);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if constexpr (sizeof(T) == 2) {
          sum = dot8(u[i], v[i], sum);
        } else {
          const float* p = reinterpret_cast<const float*>(&u[i]);
          const float* q = reinterpret_cast<const float*>(&v[i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) sum = fmaf(p[e], q[e], sum);
        }
      }
    }
  }
  for (; k < K; k += 32 * EACH) {
#pragma unroll
    for (int e = 0; e < EACH; ++e)
      if (k + e < K) sum = fmaf(fb_load_coherent(row + k + e), fb_load_coherent(w + k + e), sum);
  }
  sum = fb_warp_sum(sum);
  if (lane == 0) low[(size_t)t * rank + j] = scales[slot] * sum;
}

// out[t, n] = sum over the planes of base[., t, n] + sum_j low[t, j] B[a][n, j], a thread a feature.
template <typename T, typename Out>
__global__ void __launch_bounds__(THREADS)
adapter_expand_kernel(const float* base, int planes, long long plane_stride, long long ldb, const float* low,
                      const T* b, const int* index, int slots, int rank, int N, Out* out, long long ldo) {
  fb_pdl_wait();
  extern __shared__ __align__(16) float mine[];
  const int t = blockIdx.y, n = blockIdx.x * THREADS + threadIdx.x;
  int slot = index[t];
  if (slot >= slots) slot = -1;
  if (slot >= 0) {
    for (int j = threadIdx.x; j < rank; j += THREADS) mine[j] = __ldcg(low + (size_t)t * rank + j);
    __syncthreads();
  }
  if (n >= N) return;
  float v = 0.f;
  for (int p = 0; p < planes; ++p) v += __ldcg(base + (size_t)p * plane_stride + (size_t)t * ldb + n);
  if (slot >= 0) {
    const T* w = b + ((size_t)slot * N + n) * rank;
    float sum = 0.f;
#pragma unroll 4
    for (int j = 0; j < rank; j += 8) {  // (a multiple of 8)
      if constexpr (sizeof(T) == 2) {
        const uint4 q = ld16(w + j);
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = __bfloat1622float2(h[e]);
          sum = fmaf(mine[j + 2 * e], f.x, sum);
          sum = fmaf(mine[j + 2 * e + 1], f.y, sum);
        }
      } else {
        const uint4 q[2] = {ld16(w + j), ld16(w + j + 4)};
        const float* f = reinterpret_cast<const float*>(q);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(mine[j + e], f[e], sum);
      }
    }
    v += sum;
  }
  out[(size_t)t * ldo + n] = fb_from_float<Out>(v);
}

// ------------------------------------------------------- the other side on tensor cores
constexpr int FEATURES = 64;        // of a CTA, 16 a warp
constexpr int TOKENS = 32;
constexpr int EXPAND_THREADS = 128;
constexpr int STEPS = 8;            // k steps of 16 whose loads are on their way together

// out[t, n] = sum over the planes of base[., t, n] + sum_j low[t, j] B[a][n, j] for 32 tokens and 64
// features. The adapters of the 32 tokens come one after another, 16 ranks a step; tokens of others have
// zeros there. B comes straight from global memory: a thread takes four neighbouring ranks of a row,
// which the instruction gets as its k slots (2q, 2q + 1, 2q + 8, 2q + 9) on both sides.
template <typename Out>
__global__ void __launch_bounds__(EXPAND_THREADS)
adapter_expand_mma_kernel(const float* base, int planes, long long plane_stride, long long ldb, const float* low,
                          const __nv_bfloat16* b, const int* index, int slots, int rank, int T, int N, Out* out,
                          long long ldo) {
  extern __shared__ __align__(16) unsigned char raw[];
  float (*sums)[FEATURES + 4] = reinterpret_cast<float (*)[FEATURES + 4]>(raw);                // [TOKENS]
  __nv_bfloat16* u = reinterpret_cast<__nv_bfloat16*>(raw + TOKENS * (FEATURES + 4) * 4);      // [TOKENS][ld]
  __shared__ int s_index[TOKENS], s_slots[TOKENS], s_count;
  const int ld = rank + 8;
  fb_pdl_wait();
  fb_pdl_launch();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int t0 = blockIdx.y * TOKENS, n0 = blockIdx.x * FEATURES;
  if (warp == 0) {  // the adapters of these tokens, each once
    int slot = t0 + lane < T ? index[t0 + lane] : -1;
    if (slot >= slots) slot = -1;
    s_index[lane] = slot;
    const unsigned same = __match_any_sync(0xffffffffu, slot);
    const bool first = slot >= 0 && __ffs(same) - 1 == lane;
    const unsigned firsts = __ballot_sync(0xffffffffu, first);
    if (first) s_slots[__popc(firsts & ((1u << lane) - 1))] = slot;
    if (lane == 0) s_count = __popc(firsts);
  }
  __syncthreads();
  for (int i = tid; i < TOKENS * (rank / 4); i += EXPAND_THREADS) {
    const int t = i / (rank / 4), j = i % (rank / 4) * 4;
    if (s_index[t] < 0) continue;  // (no adapter takes its row)
    const float4 f = __ldcg(reinterpret_cast<const float4*>(low + (size_t)(t0 + t) * rank + j));
    __nv_bfloat162* to = reinterpret_cast<__nv_bfloat162*>(u + t * ld + j);
    to[0] = __floats2bfloat162_rn(f.x, f.y);
    to[1] = __floats2bfloat162_rn(f.z, f.w);
  }
  __syncthreads();
  float acc[TOKENS / 8][4];
#pragma unroll
  for (int n = 0; n < TOKENS / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  const int row0 = min(n0 + warp * 16 + g, N - 1), row1 = min(n0 + warp * 16 + g + 8, N - 1);
  const int per = (rank + 15) / 16, steps = s_count * per;
  for (int s0 = 0; s0 < steps; s0 += STEPS) {
    uint2 w[STEPS][2];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int e = (s0 + i) / per, k = (s0 + i - e * per) * 16 + 4 * q;
      w[i][0] = w[i][1] = make_uint2(0u, 0u);
      if (s0 + i < steps && k < rank) {
        const __nv_bfloat16* from = b + (size_t)s_slots[e] * N * rank + k;
        w[i][0] = __ldcg(reinterpret_cast<const uint2*>(from + (size_t)row0 * rank));
        w[i][1] = __ldcg(reinterpret_cast<const uint2*>(from + (size_t)row1 * rank));
      }
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      if (s0 + i >= steps) break;
      const int e = (s0 + i) / per, k = (s0 + i - e * per) * 16 + 4 * q, slot = s_slots[e];
#pragma unroll
      for (int n = 0; n < TOKENS / 8; ++n) {
        const int t = n * 8 + g;
        uint2 v = make_uint2(0u, 0u);
        if (s_index[t] == slot && k < rank) v = *reinterpret_cast<const uint2*>(u + t * ld + k);
        mma_bf16(acc[n], w[i][0].x, w[i][1].x, w[i][0].y, w[i][1].y, v.x, v.y);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < TOKENS / 8; ++n) {
    sums[n * 8 + 2 * q][warp * 16 + g] = acc[n][0];
    sums[n * 8 + 2 * q + 1][warp * 16 + g] = acc[n][1];
    sums[n * 8 + 2 * q][warp * 16 + g + 8] = acc[n][2];
    sums[n * 8 + 2 * q + 1][warp * 16 + g + 8] = acc[n][3];
  }
  __syncthreads();
  const bool four = (((uintptr_t)base | (uintptr_t)out) % 16) == 0 && ldb % 4 == 0 && plane_stride % 4 == 0 &&
                    ldo % 4 == 0 && n0 + FEATURES <= N;
  if (four) {
    constexpr int GROUPS = FEATURES / 4;
#pragma unroll
    for (int i0 = 0; i0 < TOKENS * GROUPS; i0 += EXPAND_THREADS) {
      const int t = (i0 + tid) / GROUPS, f = (i0 + tid) % GROUPS * 4;
      if (t0 + t >= T) continue;
      float4 v = *reinterpret_cast<const float4*>(&sums[t][f]);
      for (int p = 0; p < planes; ++p) {
        const float4 o = __ldcg(reinterpret_cast<const float4*>(base + (size_t)p * plane_stride + (size_t)(t0 + t) * ldb + n0 + f));
        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
      }
      Out* to = out + (size_t)(t0 + t) * ldo + n0 + f;
      if constexpr (sizeof(Out) == 4) {
        *reinterpret_cast<float4*>(to) = v;
      } else {
        uint2 pk;
        const __nv_bfloat162 h0 = __floats2bfloat162_rn(v.x, v.y), h1 = __floats2bfloat162_rn(v.z, v.w);
        pk.x = *reinterpret_cast<const uint32_t*>(&h0);
        pk.y = *reinterpret_cast<const uint32_t*>(&h1);
        *reinterpret_cast<uint2*>(to) = pk;
      }
    }
    return;
  }
  for (int i = tid; i < TOKENS * FEATURES; i += EXPAND_THREADS) {
    const int t = i / FEATURES, f = i % FEATURES;
    if (t0 + t >= T || n0 + f >= N) continue;
    float v = sums[t][f];
    for (int p = 0; p < planes; ++p) v += __ldcg(base + (size_t)p * plane_stride + (size_t)(t0 + t) * ldb + n0 + f);
    out[(size_t)(t0 + t) * ldo + n0 + f] = fb_from_float<Out>(v);
  }
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
  const dim3 grid((rank + THREADS / 32 - 1) / (THREADS / 32), T);
  FB_DISPATCH_DTYPE(dtype, E, fb_launch(adapter_shrink_kernel<E>, grid, dim3(THREADS), 0, stream, (const E*)x,
                                        ldx, (const E*)a, scales, index, slots, rank, K, wide, low));
  return fb_check_launch("adapter_shrink");
}

FB_API int fb_adapter_expand(const float* base, int planes, long long plane_stride, long long ldb,
                             const float* low, const void* b, int dtype, const int* index, int slots, int rank,
                             int T, int N, void* out, int out_dtype, long long ldo, cudaStream_t stream) {
  FB_REQUIRE(T >= 0 && N > 0 && rank > 0 && rank <= 1024 && rank % 8 == 0 && slots > 0 && planes > 0 &&
                 ldb >= N && ldo >= N && ((uintptr_t)b % 16) == 0,
             "adapter_expand: bad sizes T=%d N=%d rank=%d, or B not on a 16-byte boundary", T, N, rank);
  FB_REQUIRE(T <= 65535, "adapter_expand: %d tokens (65535 at most)", T);
  if (T == 0) return 0;
  const dim3 grid((N + THREADS - 1) / THREADS, T);
  FB_DISPATCH_DTYPE(dtype, E, FB_DISPATCH_DTYPE(out_dtype, O,
      fb_launch(adapter_expand_kernel<E, O>, grid, dim3(THREADS), (size_t)rank * 4, stream, base, planes,
                plane_stride, ldb, low, (const E*)b, index, slots, rank, N, (O*)out, ldo)));
  return fb_check_launch("adapter_expand");
}

// As fb_adapter_expand for bfloat16 adapters, on the tensor cores.
FB_API int fb_adapter_expand_mma(const float* base, int planes, long long plane_stride, long long ldb,
                                 const float* low, const void* b, const int* index, int slots, int rank, int T,
                                 int N, void* out, int out_dtype, long long ldo, cudaStream_t stream) {
  FB_REQUIRE(T > 0 && N > 0 && rank > 0 && rank <= 512 && rank % 8 == 0 && slots > 0 && planes > 0 && ldb >= N &&
                 ldo >= N && (((uintptr_t)b | (uintptr_t)low) % 16) == 0,
             "adapter_expand_mma: bad sizes T=%d N=%d rank=%d, or operands not on 16-byte boundaries", T, N, rank);
  FB_REQUIRE((T + TOKENS - 1) / TOKENS <= 65535, "adapter_expand_mma: %d tokens", T);
  const size_t shared = TOKENS * (FEATURES + 4) * 4 + (size_t)TOKENS * (rank + 8) * 2;  // (42 KB at rank 512)
  const dim3 grid((N + FEATURES - 1) / FEATURES, (T + TOKENS - 1) / TOKENS);
  FB_DISPATCH_DTYPE(out_dtype, O,
      fb_launch(adapter_expand_mma_kernel<O>, grid, dim3(EXPAND_THREADS), shared, stream, base, planes,
                plane_stride, ldb, low, (const __nv_bfloat16*)b, index, slots, rank, T, N, (O*)out, ldo));
  return fb_check_launch("adapter_expand_mma");
}
