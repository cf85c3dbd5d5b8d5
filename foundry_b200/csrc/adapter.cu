// Low-rank adapters of many requests beside one shared projection:
//   y[t] = x[t] W^T + scale_a (x[t] A_a^T) B_a^T,   a = index[t]  (outside of the bank: x[t] W^T)
// with A [slots, rank, K] and B [slots, N, rank] as stored. The shared product is the library's own and
// leaves 32-bit sums; `adapter_shrink` makes the rank numbers of every token, in 32 bits, and
// `adapter_expand` adds their product with B to the sums and rounds once.
#include "common.cuh"

namespace {

constexpr int THREADS = 256;

// Block t: low[t, j] = scale * sum_k x[t, k] A[a][j, k], a warp a rank.
template <typename T>
__global__ void __launch_bounds__(THREADS)
adapter_shrink_kernel(const T* x, long long ldx, const T* __restrict__ a, const float* __restrict__ scales,
                      const int* index, int slots, int rank, int K, float* low) {
  fb_pdl_wait();
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = index[t];
  if (slot < 0 || slot >= slots) return;
  const T* row = x + (size_t)t * ldx;
  for (int j = warp; j < rank; j += THREADS / 32) {
    const T* w = a + ((size_t)slot * rank + j) * K;
    float sum = 0.f;
    for (int k = lane; k < K; k += 32) sum = fmaf(fb_load_coherent(row + k), fb_to_float(w[k]), sum);
    sum = fb_warp_sum(sum);
    if (lane == 0) low[(size_t)t * rank + j] = scales[slot] * sum;
  }
}

// out[t, n] = sum over the planes of base[., t, n] + sum_j low[t, j] B[a][n, j]
template <typename T, typename Out>
__global__ void __launch_bounds__(THREADS)
adapter_expand_kernel(const float* base, int planes, long long plane_stride, long long ldb, const float* low,
                      const T* __restrict__ b, const int* index, int slots, int rank, int N, Out* out,
                      long long ldo) {
  fb_pdl_wait();
  extern __shared__ float mine[];
  const int t = blockIdx.y, n = blockIdx.x * THREADS + threadIdx.x;
  int slot = index[t];
  if (slot >= slots) slot = -1;
  if (slot >= 0) {
    for (int j = threadIdx.x; j < rank; j += THREADS) mine[j] = low[(size_t)t * rank + j];
    __syncthreads();
  }
  if (n >= N) return;
  float v = 0.f;
  for (int p = 0; p < planes; ++p) v += base[(size_t)p * plane_stride + (size_t)t * ldb + n];
  if (slot >= 0) {
    const T* w = b + ((size_t)slot * N + n) * rank;
    float sum = 0.f;
    for (int j = 0; j < rank; ++j) sum = fmaf(mine[j], fb_to_float(w[j]), sum);
    v += sum;
  }
  out[(size_t)t * ldo + n] = fb_from_float<Out>(v);
}
}  // namespace

FB_API int fb_adapter_shrink(const void* x, long long ldx, int dtype, const void* a, const float* scales,
                             const int* index, int slots, int rank, int T, int K, float* low,
                             cudaStream_t stream) {
  FB_REQUIRE(T >= 0 && K > 0 && rank > 0 && slots > 0 && ldx >= K, "adapter_shrink: bad sizes T=%d K=%d rank=%d", T,
             K, rank);
  if (T == 0) return 0;
  FB_DISPATCH_DTYPE(dtype, E, fb_launch(adapter_shrink_kernel<E>, dim3(T), dim3(THREADS), 0, stream, (const E*)x,
                                        ldx, (const E*)a, scales, index, slots, rank, K, low));
  return fb_check_launch("adapter_shrink");
}

FB_API int fb_adapter_expand(const float* base, int planes, long long plane_stride, long long ldb,
                             const float* low, const void* b, int dtype, const int* index, int slots, int rank,
                             int T, int N, void* out, int out_dtype, long long ldo, cudaStream_t stream) {
  FB_REQUIRE(T >= 0 && N > 0 && rank > 0 && rank <= 1024 && slots > 0 && planes > 0 && ldb >= N && ldo >= N,
             "adapter_expand: bad sizes T=%d N=%d rank=%d", T, N, rank);
  FB_REQUIRE(T <= 65535, "adapter_expand: %d tokens (65535 at most)", T);
  if (T == 0) return 0;
  const dim3 grid((N + THREADS - 1) / THREADS, T);
  FB_DISPATCH_DTYPE(dtype, E, FB_DISPATCH_DTYPE(out_dtype, O,
      fb_launch(adapter_expand_kernel<E, O>, grid, dim3(THREADS), (size_t)rank * 4, stream, base, planes,
                plane_stride, ldb, low, (const E*)b, index, slots, rank, N, (O*)out, ldo)));
  return fb_check_launch("adapter_expand");
}
