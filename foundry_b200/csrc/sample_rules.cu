// The draw of a row's next token under its own rules, from its edited logits (logit_edits.cuh).
//
// With v the edited logits and M their maximum (NaN counts as -inf):
//   temperature 0: the lowest index of M;
//   temperature T: tokens stand in the order (v descending, index ascending); top_k keeps the first k,
//   top_p of those the shortest prefix whose share of their sum of exp((v - M) / T) reaches p, min_p
//   those with exp((v - M) / T) >= min_p (the first one always stays); of the kept ones the largest
//   (v - M) / T + g wins, g = -log(-log u) with u of (stream, step, token) as in sampling.cu, which
//   draws from their softmax without a cumulative sum.
// The log-probability is the token's under softmax(v / T) of ALL tokens (T = 0: T = 1). A row in which
// nothing is left (every v is -inf) gives token -1 and -inf.
//
// Both borders are cuts in one order: token i of value v has the 52-bit place
// (ordered bits of v) << 20 | (2^20 - 1 - i), larger = earlier, and a cut keeps the places >= cut.
#include "logit_edits.cuh"

namespace {

constexpr int THREADS = 512;
constexpr int MAX_CLUSTER = 8;
constexpr int MAX_CHUNK = 49152;  // a block's logits in shared memory: 192 KB
constexpr unsigned ID_BITS = 20, ID_MASK = (1u << ID_BITS) - 1;

struct SampleArgs {
  const float* logits;
  long long row_stride;
  int V, chunk;
  const float* temperature;  // null: 0
  const int* top_k;          // null or <= 0: off
  const float* top_p;        // null or >= 1: off
  const float* min_p;        // null or <= 0: off
  const long long* streams;  // null: 0
  const long long* steps;
  const int* record;         // null, or a token a row that goes into its history first
  int* out;
  float* logprobs;
  int* also;                 // null, or a second place for the tokens (0 where there is none)
  FbLogitEdits edits;
};

__device__ __forceinline__ unsigned long long mix64(unsigned long long z) {
  // the SplitMix64 finaliser, as in sampling.cu
  z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ULL;
  z = (z ^ (z >> 27)) * 0x94d049bb133111ebULL;
  return z ^ (z >> 31);
}
constexpr unsigned long long GOLDEN = 0x9e3779b97f4a7c15ULL;

// -log(-log u). (z >> 40) + 0.5 has 25 bits, and the largest rounds u to one, whose noise would be
// infinite: any token would win with it. u stays below one.
__device__ __forceinline__ float gumbel(unsigned long long of_step, unsigned i) {
  const unsigned long long z = mix64(of_step + GOLDEN * ((unsigned long long)i + 1));
  const float u = fminf(((float)(unsigned)(z >> 40) + 0.5f) * (1.0f / 16777216.0f), 1.0f - 0x1p-24f);
  return -logf(-logf(u));
}

__device__ __forceinline__ unsigned ordered(float v) {
  const unsigned b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long place_of(float v, unsigned i) {
  return ((unsigned long long)ordered(v) << ID_BITS) | (ID_MASK - i);
}

__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}
__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void store_at(unsigned long long* mine, unsigned rank, unsigned long long v) {
  unsigned there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(there) : "r"((unsigned)__cvta_generic_to_shared(mine)), "r"(rank));
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(there), "l"(v) : "memory");
}

// What the blocks of a cluster tell each other: two sets by turns, so that a set is written again only
// when every block has passed the barrier behind its last reading.
struct Meeting {
  unsigned long long said[2][MAX_CLUSTER];
  unsigned long long warps[THREADS / 32];
};

template <typename F>
__device__ __forceinline__ unsigned long long meet(Meeting& m, int& turn, int blocks, unsigned rank,
                                                   unsigned long long v, F&& join) {
  // one value a thread -> one a row, joined in a fixed order, for every thread of the cluster
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) m.warps[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    v = m.warps[threadIdx.x & (THREADS / 32 - 1)];
#pragma unroll
    for (int o = THREADS / 64; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((int)threadIdx.x < blocks) store_at(&m.said[turn][rank], threadIdx.x, v);
  }
  cluster_sync();
  v = m.said[turn][0];
  for (int b = 1; b < blocks; ++b) v = join(v, m.said[turn][b]);
  turn ^= 1;
  return v;
}
struct Larger {
  __device__ unsigned long long operator()(unsigned long long a, unsigned long long b) const { return a > b ? a : b; }
};
struct Sum {
  __device__ unsigned long long operator()(unsigned long long a, unsigned long long b) const { return a + b; }
};
struct SumDoubles {
  __device__ unsigned long long operator()(unsigned long long a, unsigned long long b) const {
    return (unsigned long long)__double_as_longlong(__longlong_as_double((long long)a) +
                                                    __longlong_as_double((long long)b));
  }
};

// A row by a cluster of `gridDim.z` blocks, each with `chunk` of its logits in shared memory.
__global__ void __launch_bounds__(THREADS)
sample_rules_kernel(const SampleArgs a) {
  cluster_arrive();  // waited for in front of the first word to another block: it has to be there
  fb_pdl_wait();
  extern __shared__ __align__(16) float values[];
  __shared__ Meeting m;
  int turn = 0;
  const int blocks = (int)gridDim.z, r = blockIdx.x, tid = threadIdx.x;
  const unsigned rank = cluster_rank();
  const int lo = (int)rank * a.chunk, hi = min(a.V, lo + a.chunk), mine = max(0, hi - lo);
  const FbRowEdits row = fb_row_edits(a.edits, r, a.V);
  const float* from = a.logits + (size_t)r * a.row_stride;
  if (a.record != nullptr && row.counts != nullptr) {  // the block whose chunk holds the token
    const int t = a.record[r];
    if (t >= lo && t < hi && tid == 0) {
      row.counts[t] += 1;
      row.seen[t >> 5] |= 1u << (t & 31);
    }
    __syncthreads();
  }
  for (int i = tid; i < mine; i += THREADS) {
    float v = from[lo + i];
    if (row.counts != nullptr && (row.seen[(lo + i) >> 5] >> ((lo + i) & 31) & 1u))
      v = fb_penalised(row, v, row.counts[lo + i]);
    values[i] = v;
  }
  __syncthreads();
  fb_add_biases(a.edits, row, values, lo, hi);
  __syncthreads();
  unsigned long long first = 0;  // the first place of all: the greedy choice
  for (int i = tid; i < mine; i += THREADS) {
    float v = values[i] + 0.0f;  // no negative zero: equal values are equal places
    const bool allowed = row.allowed == nullptr || (row.allowed[(lo + i) >> 5] >> ((lo + i) & 31) & 1u);
    if (!allowed || v != v) v = -INFINITY;
    values[i] = v;
    const unsigned long long p = place_of(v, (unsigned)(lo + i));
    first = p > first ? p : first;
  }
  cluster_wait();
  first = meet(m, turn, blocks, rank, first, Larger{});
  const unsigned first_bits = (unsigned)(first >> ID_BITS);
  const float M = __uint_as_float((first_bits & 0x80000000u) ? first_bits & 0x7fffffffu : ~first_bits);
  const float T = a.temperature != nullptr ? a.temperature[r] : 0.f;
  const bool greedy = !(T > 0.f);
  const float inv_t = greedy ? 1.f : 1.0f / T;
  if (M == -INFINITY) {  // (the whole cluster)
    if (rank == 0 && tid == 0) {
      a.out[r] = -1;
      a.logprobs[r] = -INFINITY;
      if (a.also != nullptr) a.also[r] = 0;
    }
    cluster_sync();
    return;
  }
  auto shifted = [&](float v) { return v == M ? 0.f : (v - M) * inv_t; };  // (M may be +inf)
  // sum over the places from `cut` on
  auto weight_from = [&](unsigned long long cut) {
    double sum = 0.0;
    for (int i = tid; i < mine; i += THREADS)
      if (place_of(values[i], (unsigned)(lo + i)) >= cut) sum += (double)expf(shifted(values[i]));
    return __longlong_as_double((long long)meet(m, turn, blocks, rank,
                                                (unsigned long long)__double_as_longlong(sum), SumDoubles{}));
  };
  const double all = weight_from(0);
  unsigned long long best = first;
  if (!greedy) {
    unsigned long long cut = 0;
    const int k = a.top_k != nullptr ? a.top_k[r] : 0;
    if (k > 0 && k < a.V) {  // the largest cut that keeps k
      for (int bit = 31 + ID_BITS; bit >= 0; --bit) {
        const unsigned long long at = cut | (1ull << bit);
        unsigned long long count = 0;
        for (int i = tid; i < mine; i += THREADS) count += place_of(values[i], (unsigned)(lo + i)) >= at;
        if (meet(m, turn, blocks, rank, count, Sum{}) >= (unsigned long long)k) cut = at;
      }
    }
    const float p = a.top_p != nullptr ? a.top_p[r] : 1.f;
    if (p < 1.f) {  // the largest cut whose sum reaches the share
      const double share = (double)p * weight_from(cut);
      unsigned long long found = 0;
      for (int bit = 31 + ID_BITS; bit >= 0; --bit) {
        const unsigned long long at = found | (1ull << bit);
        if (weight_from(at) >= share) found = at;
      }
      cut = found > cut ? found : cut;
      cut = cut < first ? cut : first;  // a share of nothing
    }
    const float least = a.min_p != nullptr ? a.min_p[r] : 0.f;
    const unsigned long long stream = a.streams != nullptr ? (unsigned long long)a.streams[r] : 0ULL;
    const unsigned long long step = a.steps != nullptr ? (unsigned long long)a.steps[r] : 0ULL;
    const unsigned long long of_step = mix64(stream + GOLDEN * (step + 1));
    best = 0;
    for (int i = tid; i < mine; i += THREADS) {
      const float v = values[i];
      const unsigned long long at = place_of(v, (unsigned)(lo + i));
      if (at < cut || v == -INFINITY) continue;
      const float z = shifted(v);
      if (!(expf(z) >= least) && at != first) continue;
      const unsigned long long score = place_of(z + gumbel(of_step, (unsigned)(lo + i)), (unsigned)(lo + i));
      best = score > best ? score : best;
    }
    best = meet(m, turn, blocks, rank, best, Larger{});
  }
  const int token = (int)(ID_MASK - (unsigned)(best & ID_MASK));
  if (tid == 0 && token >= lo && token < hi) {
    a.out[r] = token;
    if (a.also != nullptr) a.also[r] = token;
    a.logprobs[r] = (float)((double)shifted(values[token - lo]) - log(all));
  }
  cluster_sync();  // nobody's words are still on their way to a block that has left
}
}  // namespace

// Rows of `logits` [n, V] float32 -> a token (int32) and its log-probability a row. `edits`: as for
// fb_edit_logits, or null; `record` (or null): a token a row, which its history counts as generated
// before anything is read of it. No two rows may have the same history then.
FB_API int fb_sample_rules(const float* logits, long long row_stride, int n, int V,
                           const float* temperature, const int* top_k, const float* top_p,
                           const float* min_p, const long long* streams, const long long* steps,
                           const long long* edits, const int* record, int* out, float* logprobs,
                           int* also, cudaStream_t stream) {
  FB_REQUIRE(n >= 0 && V > 0 && row_stride >= V, "sample_rules: bad sizes n=%d V=%d", n, V);
  FB_REQUIRE(V <= MAX_CLUSTER * MAX_CHUNK, "sample_rules: %d tokens (a vocabulary of %d at most)", V,
             MAX_CLUSTER * MAX_CHUNK);
  SampleArgs a{};
  a.edits = fb_unpack_edits(edits);
  if (int rc = fb_check_edits("sample_rules", a.edits, V)) return rc;
  FB_REQUIRE(record == nullptr || a.edits.counts != nullptr, "sample_rules: tokens to record, and no history");
  if (n == 0) return 0;
  int blocks = 1;
  while (blocks < MAX_CLUSTER && V > 4096 * blocks) blocks *= 2;
  a.logits = logits; a.row_stride = row_stride; a.V = V;
  a.chunk = ((V + blocks - 1) / blocks + 31) / 32 * 32;  // whole words of the bits
  a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p;
  a.streams = streams; a.steps = steps; a.record = record;
  a.out = out; a.logprobs = logprobs; a.also = also;
  static bool seen[64] = {};
  if (fb_first_use_on_device(seen)) {
    cudaError_t e = cudaFuncSetAttribute(sample_rules_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         MAX_CHUNK * 4);
    if (e != cudaSuccess) return fb_fail(2, "sample_rules: shared memory opt-in: %s", cudaGetErrorString(e));
  }
  fb_launch_cluster(sample_rules_kernel, dim3(n, 1, blocks), dim3(THREADS), (size_t)a.chunk * 4, stream,
                    (unsigned)blocks, a);
  return fb_check_launch("sample_rules");
}
