// Low-rank adapters of many requests beside one shared projection:
//   y[t] = x[t] W^T + scale_a (x[t] A_a^T) B_a^T,   a = index[t]  (outside of the bank: x[t] W^T)
// with A [slots, rank, K] and B [slots, N, rank] as stored.
//
// What it has to read beside the projection is small (a rank of 16 beside 4,096 -> 4,096: 1/128 of W for
// every adapter in the step), so what counts is that the projection's kernels run as they do without it.
//   More than 16 tokens, bfloat16: `adapter_planes` makes the rank numbers of each block of 256 tokens, a
//   plane for every adapter that has tokens in the block (zero in the rows of others), and the paired
//   tcgen05 product takes them as more K behind its own, [x | planes] [W | B]^T: one sum in tensor
//   memory, one rounding (gemm_tcgen05_pair.cu, MoreK). The rank numbers are rounded to bfloat16 for
//   that, 2^-9 of the adapter's part on average.
//   Else: `adapter_shrink` makes a token's rank numbers in 32 bits, the projection leaves 32-bit sums
//   (planes), and `adapter_expand` adds up planes and adapter and rounds once.
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

// ------------------------------------------------------------ the planes of a block
constexpr int BLOCK_ROWS = 256;  // tokens of a block: a tile of the paired product
constexpr int TOKENS = 32;       // tokens of a CTA
constexpr int RANKS = 64;        // ranks of a turn
constexpr int WARPS = THREADS / 32;
constexpr int MAX_SLOTS = 1024;
constexpr int CHUNK = 64;

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_peer(const float* mine, unsigned rank) {
  unsigned there;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(there) : "r"((unsigned)__cvta_generic_to_shared(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
  return v;
}

struct PlaneShared {
  unsigned present[MAX_SLOTS / 32];
  int slot, count, any;
  int index[TOKENS];
  float part[RANKS][TOKENS + 1];          // this CTA's share of K
  float warps[WARPS][RANKS][TOKENS + 1];  // each warp's
};

// CTA (i, e, z): of 32 tokens, the rank numbers of the e-th adapter of their block, zero in the rows of
// others; K is split over the warps and over the z CTAs of a cluster, which read each other's sums in
// order. Rows of A are the instruction's 16 rows, tokens its 8 columns, and both come straight from
// global memory in the order that the instruction wants (a thread has 16 neighbouring elements of K, as
// in gemm_skinny.cu): every warp has other bytes, so shared memory would not save any.
__global__ void __launch_bounds__(THREADS)
adapter_planes_kernel(const __nv_bfloat16* x, long long ldx, const __nv_bfloat16* a, const float* scales,
                      const int* index, int slots, int rank, int T, int K, int most, __nv_bfloat16* u,
                      int* counts, int* slots_of) {
  extern __shared__ __align__(16) unsigned char raw[];
  PlaneShared& s = *reinterpret_cast<PlaneShared*>(raw);
  fb_pdl_wait();
  fb_pdl_launch();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int t0 = blockIdx.x * TOKENS, block = t0 / BLOCK_ROWS, e = blockIdx.y;
  const int shares = gridDim.z, share = blockIdx.z;
  for (int i = tid; i < MAX_SLOTS / 32; i += THREADS) s.present[i] = 0u;
  if (tid == 0) s.any = 0;
  __syncthreads();
  {
    const int t = block * BLOCK_ROWS + tid;  // (THREADS tokens of the block)
    int slot = t < T ? index[t] : -1;
    if (slot >= slots) slot = -1;
    if (slot >= 0) atomicOr(&s.present[slot >> 5], 1u << (slot & 31));
    const int here = t - t0;
    if (here >= 0 && here < TOKENS) s.index[here] = slot;
  }
  __syncthreads();
  if (warp == 0) {  // the e-th adapter of the block, by its slot
    const unsigned word = s.present[lane];
    unsigned upto = __popc(word);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
    if (lane == 31) s.count = (int)upto;
    const int before = (int)upto - __popc(word);
    if (e >= before && e < (int)upto) s.slot = lane * 32 + (int)__fns(word, 0, e - before + 1);
  }
  __syncthreads();
  const bool tells = t0 % BLOCK_ROWS == 0 && share == 0 && tid == 0;
  if (tells && e == 0) counts[block] = s.count;
  if (e >= s.count) return;  // (every CTA of the cluster)
  const int slot = s.slot;
  if (tells) slots_of[block * most + e] = slot;
  __nv_bfloat16* rows = u + ((size_t)(block * most + e) * BLOCK_ROWS + t0 % BLOCK_ROWS) * rank;
  if (tid < TOKENS && s.index[tid] == slot) s.any = 1;
  __syncthreads();
  if (s.any == 0) {  // none of these tokens: zeros
    if (share == 0)
      for (int i = tid; i < TOKENS * rank / 8; i += THREADS)
        reinterpret_cast<uint4*>(rows)[i] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const float scale = scales[slot];
  const int chunks = (K + CHUNK - 1) / CHUNK;
  const int each = (chunks + shares * WARPS - 1) / (shares * WARPS);
  const int c0 = (share * WARPS + warp) * each, c1 = min(chunks, c0 + each);
  const __nv_bfloat16* xr[TOKENS / 8];
#pragma unroll
  for (int n = 0; n < TOKENS / 8; ++n) xr[n] = x + (size_t)min(t0 + n * 8 + g, T - 1) * ldx + q * 8;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int r0 = 0; r0 < rank; r0 += RANKS) {
    const int tiles = (min(RANKS, rank - r0) + 15) / 16;
    float acc[RANKS / 16][TOKENS / 8][4];
#pragma unroll
    for (int m = 0; m < RANKS / 16; ++m)
#pragma unroll
      for (int n = 0; n < TOKENS / 8; ++n) acc[m][n][0] = acc[m][n][1] = acc[m][n][2] = acc[m][n][3] = 0.f;
    for (int c = c0; c < c1; ++c) {
      const int k = c * CHUNK + q * 8;
      const bool lo = k + 8 <= K, hi = k + 40 <= K;
      uint4 b[TOKENS / 8][2];
#pragma unroll
      for (int n = 0; n < TOKENS / 8; ++n) {
        b[n][0] = lo ? ld16(xr[n] + (size_t)c * CHUNK) : zero;
        b[n][1] = hi ? ld16(xr[n] + (size_t)c * CHUNK + 32) : zero;
      }
#pragma unroll
      for (int m = 0; m < RANKS / 16; ++m) {
        if (m >= tiles) break;
        const __nv_bfloat16* w0 = a + ((size_t)slot * rank + min(r0 + m * 16 + g, rank - 1)) * K + k;
        const __nv_bfloat16* w1 = a + ((size_t)slot * rank + min(r0 + m * 16 + g + 8, rank - 1)) * K + k;
        const uint4 w[4] = {lo ? ld16(w0) : zero, hi ? ld16(w0 + 32) : zero, lo ? ld16(w1) : zero,
                            hi ? ld16(w1 + 32) : zero};
        const uint32_t* a0 = reinterpret_cast<const uint32_t*>(&w[0]);
        const uint32_t* a1 = reinterpret_cast<const uint32_t*>(&w[2]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int n = 0; n < TOKENS / 8; ++n) {
            const uint32_t* bx = reinterpret_cast<const uint32_t*>(&b[n][0]);
            mma_bf16(acc[m][n], a0[2 * i], a1[2 * i], a0[2 * i + 1], a1[2 * i + 1], bx[2 * i], bx[2 * i + 1]);
          }
      }
    }
#pragma unroll
    for (int m = 0; m < RANKS / 16; ++m) {
      if (m >= tiles) break;
#pragma unroll
      for (int n = 0; n < TOKENS / 8; ++n) {
        s.warps[warp][m * 16 + g][n * 8 + 2 * q] = acc[m][n][0];
        s.warps[warp][m * 16 + g][n * 8 + 2 * q + 1] = acc[m][n][1];
        s.warps[warp][m * 16 + g + 8][n * 8 + 2 * q] = acc[m][n][2];
        s.warps[warp][m * 16 + g + 8][n * 8 + 2 * q + 1] = acc[m][n][3];
      }
    }
    __syncthreads();
    for (int i = tid; i < tiles * 16 * TOKENS; i += THREADS) {
      const int j = i / TOKENS, t = i % TOKENS;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) v += s.warps[w][j][t];
      s.part[j][t] = v;
    }
    if (shares > 1) cluster_sync(); else __syncthreads();
    // the tokens' rows are shared by the cluster's CTAs; ranks side by side
    const int wide = min(RANKS, rank - r0), mine = TOKENS / shares;
    for (int i = tid; i < mine * wide; i += THREADS) {
      const int t = share * mine + i / wide, j = i % wide;
      float v = 0.f;
      if (shares > 1) {
        for (int z = 0; z < shares; ++z) v += ld_peer(&s.part[j][t], z);
      } else {
        v = s.part[j][t];
      }
      rows[(size_t)t * rank + r0 + j] = __float2bfloat16_rn(s.index[t] == slot ? scale * v : 0.f);
    }
    // nobody's sums are overwritten, or gone, while a peer still reads them
    if (shares > 1) cluster_sync(); else __syncthreads();
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

// u [ceil(T / 256) * most * 256, rank] bfloat16, counts [blocks], slots_of [blocks, most]: what
// fb_gemm_tc_adapted takes beside x and W. most: at least the adapters that one block of 256 tokens can
// have. shares: CTAs that split K (1, 2, 4 or 8).
FB_API int fb_adapter_planes(const void* x, long long ldx, const void* a, const float* scales, const int* index,
                             int slots, int rank, int T, int K, int most, int shares, void* u, int* counts,
                             int* slots_of, cudaStream_t stream) {
  FB_REQUIRE(T > 0 && K > 0 && rank > 0 && rank % 8 == 0 && slots > 0 && slots <= MAX_SLOTS && ldx >= K,
             "adapter_planes: bad sizes T=%d K=%d rank=%d slots=%d", T, K, rank, slots);
  FB_REQUIRE(most >= (slots < BLOCK_ROWS ? slots : BLOCK_ROWS) || most >= T, "adapter_planes: room for %d adapters a block", most);
  FB_REQUIRE(K % 8 == 0 && ldx % 8 == 0 && (((uintptr_t)x | (uintptr_t)a | (uintptr_t)u) % 16) == 0,
             "adapter_planes: K, the row stride and the operands must keep 16-byte alignment");
  FB_REQUIRE(shares == 1 || shares == 2 || shares == 4 || shares == 8, "adapter_planes: %d shares of K", shares);
  static bool seen[64] = {};
  if (fb_first_use_on_device(seen)) {
    cudaError_t e = cudaFuncSetAttribute(adapter_planes_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)sizeof(PlaneShared));
    if (e != cudaSuccess) return fb_fail(2, "adapter_planes: shared memory opt-in: %s", cudaGetErrorString(e));
  }
  // every row of every block is written, those behind the last token too: the product reads them
  const int blocks = (T + BLOCK_ROWS - 1) / BLOCK_ROWS;
  const dim3 grid(blocks * (BLOCK_ROWS / TOKENS), most < slots ? most : slots, shares);
  fb_launch_cluster(adapter_planes_kernel, grid, dim3(THREADS), sizeof(PlaneShared), stream, (unsigned)shares,
                    (const __nv_bfloat16*)x, ldx, (const __nv_bfloat16*)a, scales, index, slots, rank, T, K,
                    most, (__nv_bfloat16*)u, counts, slots_of);
  return fb_check_launch("adapter_planes");
}
