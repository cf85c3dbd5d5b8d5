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
//
// A row is read once, into the shared memory of a cluster. What bounds it is not those bytes (64 rows of
// 128,256: 34.7 MB, 5.3 us at the copy rate) but the passes over shared memory (some 100 instructions a logit
// under mixed rules) and the meetings of the cluster one after another, 1 to 1.5 us each: the maximum, the bins,
// a border, the winner. Device times in graph replays at 128,256 tokens, by rule (greedy, plain, top-k, top-p):
// one row 6.1, 7.4, 14.1, 14.4 us; 8 rows 7.7, 10.8, 19, 27; 33 rows 10.1, 15.4, 23.5, 41; 64 rows, two rounds
// of clusters, 19, 32, 51, 77. Where fewer than top_k tokens are within 32 temperatures of the best one, the border
// lies in the last bin and is found bit by bit: k = 50 at T = 0.1 240 us for one row, 690 for 64.
#include "logit_edits.cuh"

#include <cfloat>
#include <type_traits>

namespace {

constexpr int THREADS = 512;
constexpr int MAX_CLUSTER = 16;
// A block's logits in shared memory, 129 KB. With more of them in one bin the fractions of their
// weights could pass 32 bits (see Bins).
constexpr int MAX_CHUNK = 33024;
constexpr float SMALLEST_TEMPERATURE = 0x1p-120f;
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

__device__ __forceinline__ unsigned random_at(unsigned long long z) {
  z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ULL;
  return (unsigned)(((z ^ (z >> 27)) * 0x94d049bb133111ebULL) >> 32);
}
// The upper half of token i's random number; its top 24 bits are those of the number that sampling.cu
// makes (whose last exclusive-or does not reach them).
__device__ __forceinline__ unsigned random_of(unsigned long long of_step, unsigned i) {
  return random_at(of_step + GOLDEN * ((unsigned long long)i + 1));
}
// -log(-log u). 24 bits and a half are 25, and the largest rounds u to one, whose noise would be
// infinite: any token would win with it. u stays below one.
__device__ __forceinline__ float gumbel(unsigned random) {
  const float u = fminf(((float)(random >> 8) + 0.5f) * (1.0f / 16777216.0f), 1.0f - 0x1p-24f);
  return -logf(-logf(u));
}
// 2^a, within 2^-22 of it
__device__ __forceinline__ float exp2_fast(float a) {
  float v;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(v) : "f"(a));
  return v;
}

// A weight in 64 bits: it is positive or zero and no denormal number, so its bits need only be moved (zero
// becomes 2^-127, nothing beside the largest weight, which is one). The conversion runs at an eighth of the rate.
__device__ __forceinline__ double widened(float w) {
  const unsigned b = __float_as_uint(w);
  return __hiloint2double((int)((b >> 3) + (896u << 20)), (int)(b << 29));
}

__device__ __forceinline__ unsigned ordered(float v) {
  const unsigned b = __float_as_uint(v + 0.0f);  // no negative zero: equal values are equal places
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

// What the blocks of a cluster tell each other: two sets by turns, so that a set is written again only
// when every block has passed the barrier behind its last reading.
struct Meeting {
  unsigned long long said[2][2][MAX_CLUSTER];
  unsigned long long warps[2][THREADS / 32];
};

// One value a thread -> one a row, joined in a fixed order, for every thread of the cluster; `meanwhile`
// runs while the blocks wait for each other. The pair form takes two values with joins of their own.
// The join of a warp's values, for every lane. The larger of two places: their upper 32 bits, then the
// lower ones of those that have them, by the warp's own reductions.
template <int LANES, typename F>
__device__ __forceinline__ unsigned long long over_warp(unsigned long long v, F&& join) {
  if constexpr (std::is_same_v<std::remove_cv_t<std::remove_reference_t<F>>, Larger>) {
    const unsigned upper = (unsigned)(v >> ID_BITS);
    const unsigned most = __reduce_max_sync(0xffffffffu, upper);
    const unsigned lower = __reduce_max_sync(0xffffffffu, upper == most ? (unsigned)v & ID_MASK : 0u);
    return ((unsigned long long)most << ID_BITS) | lower;
  } else {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }
}

template <typename F, typename G, typename W>
__device__ __forceinline__ void meet_pair(Meeting& m, int& turn, int blocks, unsigned rank,
                                          unsigned long long& v, F&& join, unsigned long long* w, G&& join_w,
                                          W&& meanwhile) {
  v = over_warp<32>(v, join);
  if (w != nullptr) *w = over_warp<32>(*w, join_w);
  const int lane = threadIdx.x & 31;
  if (lane == 0) {
    m.warps[0][threadIdx.x >> 5] = v;
    if (w != nullptr) m.warps[1][threadIdx.x >> 5] = *w;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    v = m.warps[0][lane & (THREADS / 32 - 1)];
    if (w != nullptr) *w = m.warps[1][lane & (THREADS / 32 - 1)];
    v = over_warp<THREADS / 32>(v, join);
    if (w != nullptr) *w = over_warp<THREADS / 32>(*w, join_w);
    if (lane < blocks) {
      store_at(&m.said[turn][0][rank], lane, v);
      if (w != nullptr) store_at(&m.said[turn][1][rank], lane, *w);
    }
  }
  cluster_arrive();
  meanwhile();
  cluster_wait();
  // every warp joins what the blocks said
  v = m.said[turn][0][lane & (blocks - 1)];
  if (w != nullptr) *w = m.said[turn][1][lane & (blocks - 1)];
  if constexpr (std::is_same_v<std::remove_cv_t<std::remove_reference_t<F>>, Larger>) {
    v = over_warp<32>(v, join);
  } else {
    for (int o = blocks / 2; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
  }
  if (w != nullptr)
    for (int o = blocks / 2; o > 0; o >>= 1) *w = join_w(*w, __shfl_xor_sync(0xffffffffu, *w, o));
  turn ^= 1;
}
template <typename F>
__device__ __forceinline__ unsigned long long meet(Meeting& m, int& turn, int blocks, unsigned rank,
                                                   unsigned long long v, F&& join) {
  meet_pair(m, turn, blocks, rank, v, join, (unsigned long long*)nullptr, join, [] {});
  return v;
}
// The border of a rule between the tokens of one bin of weights, found where it lies between too many
// equal or nearly equal ones for the list in shared memory: a bit of the place a meeting, 52 meetings.
// The largest cut for which `amount(cut)`, the cluster's sum over the bin's places >= cut, reaches `need`.
template <typename F>
__device__ __noinline__ unsigned long long cut_by_bits(F&& amount, unsigned long long need) {
  unsigned long long cut = 0;
  for (int bit = 31 + ID_BITS; bit >= 0; --bit) {
    const unsigned long long at = cut | (1ull << bit);
    if (amount(at) >= need) cut = at;
  }
  return cut;
}

// Tokens by their distance d = (M - v) / T from the best one: bins of 1 / 32, the last one for all
// that is further than 32. Inside a bin the weights exp(-d) are exp(-b / 32) (1 - part), with part below
// 0.031; its 22-bit fraction adds up as whole numbers, so that the sums do not depend on the order
// in which threads come. What the last bin weighs (V exp(-32) at most) is left out of the sums.
// Two zones, near bins and the rest, were slower (64 rows of 128,256 under every kind of rule 86 us where one zone
// took 82).
constexpr int BINS = 1024;
constexpr float BINS_PER_UNIT = 32.f;
constexpr int PART_BITS = 22;
constexpr int LISTED = 128;  // tokens of a border's bin that are compared with each other in shared memory
constexpr int SLICES = THREADS;
static_assert(LISTED * 4 == THREADS, "four threads a token of the list, or more");

// A distance in 32nds: its bin (an edge belongs to either side, always the same one), and 1 - exp(-x) of
// what is left of it, x <= 1 / 32, by its series (the next term is below 2^-31), in units of 2^-22. Whole
// numbers are made and taken off by adding 1.5 * 2^23, which leaves them in the last bits.
constexpr float TO_WHOLE = 12582912.f;
__device__ __forceinline__ bool in_last_bin(float t) { return !(t < (float)(BINS - 1)); }
__device__ __forceinline__ int bin_of(float t) {
  return in_last_bin(t) ? BINS - 1 : __float_as_int((t - 0.5f) + TO_WHOLE) & 0xffff;
}
__device__ __forceinline__ unsigned part_of(float t) {  // of a token in front of the last bin
  const float x = t - (((t - 0.5f) + TO_WHOLE) - TO_WHOLE);  // exact
  // 2^22 (y - y^2 / 2 + y^3 / 6 - y^4 / 24) at y = x / 32
  const float part = x * (131072.f - x * (2048.f - x * (64.f / 3.f - x * (1.f / 6.f))));
  return (unsigned)__float_as_int(part + TO_WHOLE) & 0x3ffffu;
}
__device__ __forceinline__ int slice_of(float t) {  // of a token in front of the last bin
  const float x = t - (((t - 0.5f) + TO_WHOLE) - TO_WHOLE);  // in [0, 1], exact
  return min(SLICES - 1, (int)(x * (float)SLICES));
}
__device__ __forceinline__ unsigned weight_in_bin(float t) {
  return in_last_bin(t) ? 0u : (1u << PART_BITS) - part_of(t);
}
__device__ __forceinline__ float value_of(unsigned long long place) {
  const unsigned bits = (unsigned)(place >> ID_BITS);
  return __uint_as_float((bits & 0x80000000u) ? bits & 0x7fffffffu : ~bits);
}

struct Bins {
  unsigned count[BINS], part[BINS];      // this block's tokens
  unsigned all_count[BINS];              // the row's
  float all_weight[BINS];
  unsigned long long listed[LISTED], own[LISTED];  // the row's, and this block's part of them
  unsigned long long scan_warps[2][THREADS / 32];
  // of each of the two borders: its bin + 1, this block's tokens in it so far, what stands in front
  unsigned found[2], counted[2], last[2], count_front[2], tokens[2], weighs[LISTED];
  double weight_front[2];
  unsigned long long cut[2];
  // the same for a border's bin cut up once more, where it holds more tokens than the list: a slice a
  // thread; weights in two halves of 11 bits, then whole
  unsigned slice_count[SLICES], slice_low[SLICES], slice_high[SLICES], all_slice_count[SLICES];
  unsigned long long all_slice_weight[SLICES], slice_weight_front[2];
  unsigned slice_found[2], slice_count_front[2];
};

template <typename T>
__device__ __forceinline__ T load_at(const T* mine, unsigned rank) {
  unsigned there, v;
  static_assert(sizeof(T) == 4, "words");
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(there) : "r"((unsigned)__cvta_generic_to_shared(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(there) : "memory");
  return (T)v;
}
__device__ __forceinline__ void store_word_at(void* mine, unsigned rank, unsigned v) {
  unsigned there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(there) : "r"((unsigned)__cvta_generic_to_shared(mine)), "r"(rank));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there), "r"(v) : "memory");
}

template <int BYTES>
__device__ __forceinline__ void copy_async(float* to, const float* from) {
  const unsigned there = (unsigned)__cvta_generic_to_shared(to);
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(there), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(there), "l"(from) : "memory");
}

// A row by a cluster of `gridDim.z` blocks, each with `chunk` of its logits in shared memory.
// AN_SM blocks of it run on an SM: alone there it may use more registers (32,000 tokens a row, top-p 12.3 us
// against 13.0 for one row, 26.2 against 27.2 for 64).
template <int AN_SM>
__global__ void __launch_bounds__(THREADS, AN_SM)
sample_rules_kernel(const SampleArgs a) {
  cluster_arrive();  // waited for in front of the first word to another block: it has to be there
  fb_pdl_wait();
  extern __shared__ __align__(16) float values[];
  Bins& bins = *reinterpret_cast<Bins*>(values + a.chunk);
  __shared__ Meeting m;
  int turn = 0;
  const int blocks = (int)gridDim.z, r = blockIdx.x, tid = threadIdx.x;
  const unsigned rank = cluster_rank();
  const int lo = (int)rank * a.chunk, hi = min(a.V, lo + a.chunk), mine = max(0, hi - lo);
  const float* from = a.logits + (size_t)r * a.row_stride + lo;
  const FbRowEdits row = fb_row_edits(a.edits, r, a.V);
  const float asked = a.temperature != nullptr ? a.temperature[r] : 0.f;
  // (an infinite one: equal shares. The smallest: 32 / T and log2(e) / T stay finite, so that the best token's lead of
  // zero is no NaN; a smaller one would draw otherwise only between logits less than 2^-113 apart.)
  const float T = asked > 0.f ? fminf(fmaxf(asked, SMALLEST_TEMPERATURE), FLT_MAX) : 0.f;
  const bool greedy = !(T > 0.f);
  const int k = a.top_k != nullptr && !greedy ? a.top_k[r] : 0;
  const float p = a.top_p != nullptr && !greedy ? a.top_p[r] : 1.f;
  const float least = a.min_p != nullptr ? a.min_p[r] : 0.f;
  const bool cuts = (k > 0 && k < a.V) || p < 1.f;
  if (a.record != nullptr && row.counts != nullptr) {  // the block whose chunk holds the token
    const int t = a.record[r];
    if (t >= lo && t < hi && tid == 0) {
      row.counts[t] += 1;
      row.seen[t >> 5] |= 1u << (t & 31);
    }
    __syncthreads();
  }
  const bool biased = row.bias_from < row.bias_to;
  // The logits go to shared memory as they are, all asked for at once (loads into registers took a trip to
  // memory for every 8,192 of a block). Meanwhile the places of the history's tokens are put on a list (in the
  // bins' room, which nobody needs yet), which the block's threads then work off, one load of a count each, all
  // at once (logit_edits.cu says what that saves).
  __shared__ int hit_count;
  unsigned short* hits = reinterpret_cast<unsigned short*>(&bins);
  constexpr int MOST_HITS = sizeof(Bins) / 2;
  int done = 0;
  if ((reinterpret_cast<uintptr_t>(from) & 15) == 0) {
    done = mine & ~3;
    for (int i = 4 * tid; i < done; i += 4 * THREADS) copy_async<16>(values + i, from + i);
  }
  for (int i = done + tid; i < mine; i += THREADS) copy_async<4>(values + i, from + i);
  // what is looked at four by four ends with tokens that have no chance
  const int padded = (mine + 3) & ~3;
  if (mine + tid < padded) values[mine + tid] = -INFINITY;
  const unsigned* allowed = row.allowed != nullptr ? row.allowed + (lo >> 5) : nullptr;
  if (row.counts != nullptr) {
    if (tid == 0) hit_count = 0;
    __syncthreads();
    for (int w = tid; 32 * w < mine; w += THREADS) {
      unsigned held = row.seen[(lo >> 5) + w];
      if (mine - 32 * w < 32) held &= (1u << (mine - 32 * w)) - 1;
      if (held == 0u) continue;
      int at = atomicAdd(&hit_count, __popc(held));
      for (; held != 0u && at < MOST_HITS; held &= held - 1, ++at) hits[at] = (unsigned short)(32 * w + __ffs(held) - 1);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  if (row.counts != nullptr) {
    auto penalise = [&](int i) { values[i] = fb_penalised(row, values[i], row.counts[lo + i]); };
    if (hit_count <= MOST_HITS) {
      for (int i = tid; i < hit_count; i += THREADS) penalise(hits[i]);
    } else {  // (the list has no room for so many)
      for (int i = tid; i < mine; i += THREADS)
        if (row.seen[(lo + i) >> 5] >> (i & 31) & 1u) penalise(i);
    }
    __syncthreads();
  }
  if (biased) {
    fb_add_biases(a.edits, row, values, lo, hi);
    __syncthreads();
  }
  // NaN has no chance, like a token that is not allowed
  float top = -INFINITY;  // the thread's best value
  if (allowed != nullptr) {
#pragma unroll 2
    for (int i = 4 * tid; i < padded; i += 4 * THREADS) {
      float4 f = *reinterpret_cast<float4*>(values + i);
      const unsigned ok = allowed[i >> 5] >> (i & 31);
      f.x = ok & 1u ? fmaxf(f.x, -INFINITY) : -INFINITY;
      f.y = ok & 2u ? fmaxf(f.y, -INFINITY) : -INFINITY;
      f.z = ok & 4u ? fmaxf(f.z, -INFINITY) : -INFINITY;
      f.w = ok & 8u ? fmaxf(f.w, -INFINITY) : -INFINITY;
      top = fmaxf(fmaxf(top, fmaxf(f.x, f.y)), fmaxf(f.z, f.w));
      *reinterpret_cast<float4*>(values + i) = f;
    }
  } else {
#pragma unroll 2
    for (int i = 4 * tid; i < padded; i += 4 * THREADS) {
      float4 f = *reinterpret_cast<float4*>(values + i);
      if (isnan((f.x + f.y) + (f.z + f.w))) {  // (or infinities of both signs)
        f.x = fmaxf(f.x, -INFINITY);
        f.y = fmaxf(f.y, -INFINITY);
        f.z = fmaxf(f.z, -INFINITY);
        f.w = fmaxf(f.w, -INFINITY);
        *reinterpret_cast<float4*>(values + i) = f;
      }
      top = fmaxf(fmaxf(top, fmaxf(f.x, f.y)), fmaxf(f.z, f.w));
    }
  }
  // where it comes first: looked for by the threads that have their warp's best value alone
  int top_at = -1;
  const unsigned top_of_warp = __reduce_max_sync(0xffffffffu, ordered(top));
  if (top > -INFINITY && ordered(top) == top_of_warp) {
    for (int i = 4 * tid; top_at < 0; i += 4 * THREADS) {
      const float4 f = *reinterpret_cast<float4*>(values + i);
      if (f.x == top) top_at = i;
      else if (f.y == top) top_at = i + 1;
      else if (f.z == top) top_at = i + 2;
      else if (f.w == top) top_at = i + 3;
    }
  }
  if (cuts) {
    for (int b = tid; b < BINS; b += THREADS) bins.count[b] = bins.part[b] = 0;
    if (tid < 2) bins.found[tid] = bins.counted[tid] = bins.last[tid] = bins.slice_found[tid] = 0;
  }
  const float inv_t = greedy ? 1.f : 1.0f / T;
  // exp(-(M - v) / T) as a power of two; the factor -log2(e) / T, log2(e) in two parts, rounded once
  float log2_t = -1.44269502f * inv_t;
  {
    const float t = greedy ? 1.f : T;
    const float q = 1.44269502f / t;
    log2_t = -(q + (fmaf(-q, t, 1.44269502f) + 1.9259630e-8f) / t);
  }
  const unsigned long long stream = a.streams != nullptr ? (unsigned long long)a.streams[r] : 0ULL;
  const unsigned long long step = a.steps != nullptr ? (unsigned long long)a.steps[r] : 0ULL;
  const unsigned long long of_step = mix64(stream + GOLDEN * (step + 1));
  cluster_wait();
  // the first place of all: the greedy choice
  unsigned long long first = top_at >= 0 ? place_of(top, (unsigned)(lo + top_at)) : 0;
  first = meet(m, turn, blocks, rank, first, Larger{});
  if (first == 0) {  // nothing is left (the whole cluster sees it)
    if (rank == 0 && tid == 0) {
      a.out[r] = -1;
      a.logprobs[r] = -INFINITY;
      if (a.also != nullptr) a.also[r] = 0;
    }
    cluster_sync();
    return;
  }
  if (value_of(first) == INFINITY) {  // infinite logits: these share all there is, equally
    for (int i = tid; i < mine; i += THREADS) values[i] = values[i] == INFINITY ? 0.f : -INFINITY;
    first = place_of(0.f, ID_MASK - (unsigned)(first & ID_MASK));
    __syncthreads();
  }
  const float M = value_of(first);
  auto weight_of = [&](float v) { return exp2_fast((M - v) * log2_t); };
  auto distance = [&](float v) { return (M - v) * inv_t; };
  const float bins_t = inv_t * BINS_PER_UNIT;
  auto binned = [&](float v) { return (M - v) * bins_t; };
  auto four_at = [&](int i) { return *reinterpret_cast<const float4*>(values + i); };
  // The winner of the draw so far, as a place of its score. A token of weight w beats score s where
  // -log u < w exp(-s), and -log u >= 1 - u: all but a few of the tokens need no logarithm (with a
  // thousandth more of the right side than rounding could ask for; 1 - u from 23 of its bits, a unit
  // less). The first token's score is where every thread starts: that one is always kept.
  const unsigned first_id = ID_MASK - (unsigned)(first & ID_MASK);
  unsigned long long best = greedy ? first : place_of(gumbel(random_of(of_step, first_id)), first_id);
  float beaten = greedy ? 0.f : 1.001f * expf(-value_of(best));
  auto may_win = [&](unsigned random, float w) {
    return (2.0f - 0x1p-22f) - __uint_as_float(random >> 9 | 0x3f800000u) <= w * beaten && w >= least;
  };
  auto try_token = [&](float v, unsigned random, unsigned id) {
    const unsigned long long score = place_of(gumbel(random) - distance(v), id);
    if (score > best) {
      best = score;
      beaten = 1.001f * expf(-value_of(best));
    }
  };
  // The best of a warp is what its other threads' tokens have to beat as well: of a flat row's tokens nearly
  // every one that a thread looks at first beats its own best so far.
  auto share_the_best = [&] { beaten = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(beaten))); };
  double all = 0.0;
  if (!cuts) {  // one pass: the sum of the weights and the draw
    if (greedy) {
#pragma unroll 2
      for (int i = 4 * tid; i < padded; i += 4 * THREADS) {
        const float4 v = four_at(i);
        all += (widened(weight_of(v.x)) + widened(weight_of(v.y))) + (widened(weight_of(v.z)) + widened(weight_of(v.w)));
      }
    } else {
      unsigned long long z = of_step + GOLDEN * ((unsigned long long)(lo + 4 * tid) + 1);
#pragma unroll 2
      for (int i0 = 0; i0 < padded; i0 += 4 * THREADS, z += 4 * THREADS * GOLDEN) {  // (whole warps)
        const int i = i0 + 4 * tid;
        const float4 f = i < padded ? four_at(i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        const float v[4] = {f.x, f.y, f.z, f.w};
        float w[4];
        unsigned random[4];
        bool any = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[j] = weight_of(v[j]);
          random[j] = random_at(z + j * GOLDEN);
          any |= may_win(random[j], w[j]);
        }
        all += (widened(w[0]) + widened(w[1])) + (widened(w[2]) + widened(w[3]));
        if (__any_sync(0xffffffffu, any)) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (may_win(random[j], w[j])) try_token(v[j], random[j], (unsigned)(lo + i + j));
          share_the_best();
        }
      }
    }
  } else {
    unsigned far = 0;
#pragma unroll 2
    for (int i = 4 * tid; i < padded; i += 4 * THREADS) {
      const float4 f = four_at(i);
      const float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float t = binned(v[j]);
        const bool near = !in_last_bin(t);
        const unsigned part = part_of(t);
        const int b = bin_of(t);
        if (near) {
          atomicAdd(&bins.count[b], 1u);
          atomicAdd(&bins.part[b], part);
        }
        far += !near && v[j] != -INFINITY;
      }
    }
    // the last bin may hold nearly all tokens: their number is made by warps
    far = __reduce_add_sync(0xffffffffu, far);
    if ((tid & 31) == 0 && far != 0) atomicAdd(&bins.count[BINS - 1], far);
    // Each block adds up its share of the bins over the cluster and tells everybody: blocks / 2 neighbouring
    // lanes a bin, each with two of the blocks (one thread a bin, asking them all in a row, took 2 us).
    const int share = BINS / blocks, lanes = max(1, blocks / 2), part_of_bin = tid & (lanes - 1);
    cluster_arrive();
    const double exact_unit = exp(-(double)((int)rank * share + tid / lanes) / BINS_PER_UNIT);
    cluster_wait();
    for (int i = tid / lanes; i < share; i += THREADS / lanes) {  // (a second round only for one block's bins)
      const int b = (int)rank * share + i;
      unsigned count = 0;
      unsigned long long part = 0;
      for (int o = part_of_bin; o < blocks; o += lanes) {
        count += load_at(&bins.count[b], o);
        part += load_at(&bins.part[b], o);
      }
      for (int o = lanes / 2; o > 0; o /= 2) {
        count += __shfl_xor_sync(0xffffffffu, count, o);
        part += __shfl_xor_sync(0xffffffffu, part, o);
      }
      const double unit = i < THREADS / lanes ? exact_unit : exp(-(double)b / BINS_PER_UNIT);
      const double size = (double)(((unsigned long long)count << PART_BITS) - part) * (1.0 / (1 << PART_BITS));
      const float weight = b == BINS - 1 ? 0.f : (float)(unit * size);
      for (int o = part_of_bin; o < blocks; o += lanes) {
        store_word_at(&bins.all_count[b], o, count);
        store_word_at(&bins.all_weight[b], o, __float_as_uint(weight));
      }
    }
    cluster_sync();
    // every block for itself from here on, with the same numbers in the same order: what stands in
    // front of each bin. A thread has BINS / THREADS bins side by side.
    constexpr int EACH = BINS / THREADS;
    unsigned counts[EACH], count_before;
    float weights[EACH];
    double weight_before;
    unsigned left = 0;  // tokens that the edits leave at all
    {
      unsigned c = 0;
      double w = 0.0;
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        counts[j] = bins.all_count[tid * EACH + j];
        weights[j] = bins.all_weight[tid * EACH + j];
        c += counts[j];
        w += (double)weights[j];
      }
      unsigned upto_c = c;
      double upto_w = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned oc = __shfl_up_sync(0xffffffffu, upto_c, o);
        const double ow = __shfl_up_sync(0xffffffffu, upto_w, o);
        if ((tid & 31) >= o) { upto_c += oc; upto_w += ow; }
      }
      if ((tid & 31) == 31) {
        bins.scan_warps[0][tid >> 5] = upto_c;
        bins.scan_warps[1][tid >> 5] = (unsigned long long)__double_as_longlong(upto_w);
      }
      __syncthreads();
      unsigned front_c = 0;
      double front_w = 0.0;
#pragma unroll
      for (int o = 0; o < THREADS / 32; ++o) {
        const unsigned oc = (unsigned)bins.scan_warps[0][o];
        const double ow = __longlong_as_double((long long)bins.scan_warps[1][o]);
        if (o < (tid >> 5)) {
          front_c += oc;
          front_w += ow;
        }
        left += oc;
        all += ow;
      }
      count_before = front_c + upto_c - c;
      weight_before = front_w + (upto_w - w);
    }
    // The border of a rule: the last bin with tokens whose front is below `target`, put in order, and
    // of its tokens the last one whose front is. Rule 0: fronts count tokens, 1: they weigh.
    double kept_sum = all;  // what the last border keeps weighs
    bool listed_before = false;
    auto border = [&](int rule, double target) -> unsigned long long {
      {
        unsigned c = count_before, at = 0;
        double w = weight_before;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
          if (counts[j] != 0 && (rule == 0 ? (double)c : w) < target) at = tid * EACH + j + 1;
          c += counts[j];
          w += (double)weights[j];
        }
        at = __reduce_max_sync(0xffffffffu, at);
        if ((tid & 31) == 0 && at != 0) atomicMax(&bins.found[rule], at);
      }
      __syncthreads();
      if (bins.found[rule] == 0) return first;  // a share of nothing
      const int b = (int)bins.found[rule] - 1;
      if (tid == b / EACH) {
        unsigned c = count_before;
        double w = weight_before;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
          if (j < b % EACH) { c += counts[j]; w += (double)weights[j]; }
        }
        bins.count_front[rule] = c;
        bins.weight_front[rule] = w;
        bins.tokens[rule] = bins.all_count[b];
      }
      // (an error of 2^-23 of what this bin weighs, and none in the first bin)
      const double unit = b == BINS - 1 ? 0.0 : (double)expf(-(float)b * (1.f / BINS_PER_UNIT)) * (1.0 / (1 << PART_BITS));
      auto fixed = [&](float v) { return weight_in_bin(binned(v)); };
      __syncthreads();
      double c_front = (double)bins.count_front[rule];
      const double w_front = bins.weight_front[rule];
      unsigned long long front_in_bin = 0;  // in units of the bin
      unsigned n = bins.tokens[rule];
      int slice = -1;
      // (values a bin further on either side than the border's bin, and what rounding could make of
      // that; most tokens lie outside)
      const float far = (float)(b + 2) / bins_t, room = 0x1p-21f * (fabsf(M) + far);
      const float v_from = b == BINS - 1 ? -INFINITY : (M - far) - room;
      const float v_to = (M - (float)(b - 1) / bins_t) + room;
      auto none_near = [&](const float (&v)[4]) {
        return !((v[0] >= v_from && v[0] <= v_to) || (v[1] >= v_from && v[1] <= v_to) ||
                 (v[2] >= v_from && v[2] <= v_to) || (v[3] >= v_from && v[3] <= v_to));
      };
      if (n > LISTED && b != BINS - 1) {  // once more, inside the bin
        bins.slice_count[tid] = bins.slice_low[tid] = bins.slice_high[tid] = 0;
        __syncthreads();
#pragma unroll 2
        for (int i = 4 * tid; i < padded; i += 4 * THREADS) {
          const float4 f = four_at(i);
          const float v[4] = {f.x, f.y, f.z, f.w};
          if (none_near(v)) continue;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float t = binned(v[j]);
            if (bin_of(t) != b) continue;
            const int at = slice_of(t);
            const unsigned w = weight_in_bin(t);
            atomicAdd(&bins.slice_count[at], 1u);
            atomicAdd(&bins.slice_low[at], w & 2047u);
            atomicAdd(&bins.slice_high[at], w >> 11);
          }
        }
        cluster_sync();
        {  // as the bins: a thread a block and a slice
          const int at = (int)rank * (SLICES / blocks) + tid / blocks, o = tid & (blocks - 1);
          unsigned count = load_at(&bins.slice_count[at], o);
          unsigned long long weight = (unsigned long long)load_at(&bins.slice_high[at], o) << 11;
          weight += load_at(&bins.slice_low[at], o);
          for (int l = blocks / 2; l > 0; l /= 2) {
            count += __shfl_xor_sync(0xffffffffu, count, l);
            weight += __shfl_xor_sync(0xffffffffu, weight, l);
          }
          store_word_at(&bins.all_slice_count[at], o, count);
          store_at(&bins.all_slice_weight[at], o, weight);
        }
        cluster_sync();
        const unsigned mine_c = bins.all_slice_count[tid];
        const unsigned long long mine_w = bins.all_slice_weight[tid];
        unsigned upto_c = mine_c;
        unsigned long long upto_w = mine_w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned oc = __shfl_up_sync(0xffffffffu, upto_c, o);
          const unsigned long long ow = __shfl_up_sync(0xffffffffu, upto_w, o);
          if ((tid & 31) >= o) { upto_c += oc; upto_w += ow; }
        }
        if ((tid & 31) == 31) {
          bins.scan_warps[0][tid >> 5] = upto_c;
          bins.scan_warps[1][tid >> 5] = upto_w;
        }
        __syncthreads();
#pragma unroll
        for (int o = 0; o < THREADS / 32; ++o) {
          if (o < (tid >> 5)) {
            upto_c += (unsigned)bins.scan_warps[0][o];
            upto_w += bins.scan_warps[1][o];
          }
        }
        upto_c -= mine_c;  // in front of this thread's slice
        upto_w -= mine_w;
        const bool in_front = rule == 0 ? c_front + (double)upto_c < target : w_front + unit * (double)upto_w < target;
        const unsigned at = __reduce_max_sync(0xffffffffu, mine_c != 0 && in_front ? tid + 1 : 0);
        if ((tid & 31) == 0 && at != 0) atomicMax(&bins.slice_found[rule], at);
        __syncthreads();
        slice = max(0, (int)bins.slice_found[rule] - 1);
        if (tid == slice) {
          bins.slice_count_front[rule] = upto_c;
          bins.slice_weight_front[rule] = upto_w;
        }
        __syncthreads();
        c_front += (double)bins.slice_count_front[rule];
        front_in_bin = bins.slice_weight_front[rule];
        n = bins.all_slice_count[slice];
      }
      auto in_border = [&](float v) {
        const float t = binned(v);
        return bin_of(t) == b && v != -INFINITY && (slice < 0 || slice_of(t) == slice);
      };
      if (n <= LISTED) {
        // everybody gets everybody's tokens of the bin; a block's stand behind those of lower ranks
        if (listed_before) cluster_sync();  // everybody is through with the list of the border before
        listed_before = true;
        const int lane = tid & 31;
        const unsigned base = __reduce_add_sync(0xffffffffu, lane < (int)rank ?
            load_at(slice < 0 ? &bins.count[b] : &bins.slice_count[slice], lane) : 0u);
#pragma unroll 2
        for (int i = 4 * tid; i < padded; i += 4 * THREADS) {
          const float4 f = four_at(i);
          const float v[4] = {f.x, f.y, f.z, f.w};
          if (none_near(v)) continue;
          bool in[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) in[j] = in_border(v[j]);
          if (in[0] || in[1] || in[2] || in[3]) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (in[j]) bins.own[atomicAdd(&bins.counted[rule], 1u)] = place_of(v[j], (unsigned)(lo + i + j));
          }
        }
        __syncthreads();
        for (unsigned i = tid; i < bins.counted[rule] * blocks; i += THREADS) {
          const unsigned k = i / blocks;
          store_at(&bins.listed[base + k], i - k * blocks, bins.own[k]);
        }
        cluster_sync();
        if (n <= 32) {  // every warp for itself: how many are in front of each, and what do they weigh
          const unsigned long long me = lane < (int)n ? bins.listed[lane] : 0ull;
          const unsigned weighs = lane < (int)n ? fixed(value_of(me)) : 0u;
          unsigned ahead = 0, in_front = 0;
          for (unsigned j = 0; j < n; ++j) {
            const unsigned long long other = __shfl_sync(0xffffffffu, me, j);
            const unsigned w = __shfl_sync(0xffffffffu, weighs, j);
            if (other > me) {
              ++ahead;
              in_front += w;
            }
          }
          const bool kept = lane < (int)n &&
              (rule == 0 ? c_front + (double)ahead : w_front + unit * (double)(front_in_bin + in_front)) < target;
          const unsigned many = __reduce_max_sync(0xffffffffu, kept ? ahead + 1 : 0u);
          const unsigned last = __ballot_sync(0xffffffffu, kept && ahead + 1 == many);
          const int who = last != 0 ? __ffs(last) - 1 : 0;
          kept_sum = w_front + unit * (double)(front_in_bin + __shfl_sync(0xffffffffu, in_front + weighs, who));
          return __shfl_sync(0xffffffffu, me, who);
        }
        // a group of neighbouring threads a token: how many are in front of it, and what do they weigh (128
        // tokens less than 2^29)
        unsigned each = THREADS / 64;  // threads a token
        while (each * n > THREADS) each /= 2;
        const unsigned who = tid / each;
        const unsigned long long me = who < n ? bins.listed[who] : 0ull;
        if (tid < (int)n) bins.weighs[tid] = fixed(value_of(bins.listed[tid]));
        __syncthreads();
        unsigned ahead = 0, in_front = 0;
#pragma unroll 4
        for (unsigned j = tid & (each - 1); j < n; j += each) {
          if (bins.listed[j] > me) {
            ++ahead;
            in_front += bins.weighs[j];
          }
        }
        for (unsigned o = each / 2; o > 0; o /= 2) {
          ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
          in_front += __shfl_xor_sync(0xffffffffu, in_front, o);
        }
        const bool kept = who < n &&
            (rule == 0 ? c_front + (double)ahead : w_front + unit * (double)(front_in_bin + in_front)) < target;
        const unsigned many = __reduce_max_sync(0xffffffffu, kept ? ahead + 1 : 0u);
        if (lane == 0 && many != 0) atomicMax(&bins.last[rule], many);
        __syncthreads();
        if (who < n && ahead + 1 == max(1u, bins.last[rule]) && (tid & (each - 1)) == 0) {
          bins.cut[rule] = me;
          bins.weight_front[rule] = w_front + unit * (double)(front_in_bin + in_front + bins.weighs[who]);
        }
        __syncthreads();
        kept_sum = bins.weight_front[rule];
        return bins.cut[rule];
      }
      auto amount = [&](unsigned long long cut, bool count) {
        unsigned long long sum = 0;
        for (int i = tid; i < mine; i += THREADS) {
          const float v = values[i];
          if (!in_border(v) || place_of(v, (unsigned)(lo + i)) < cut) continue;
          sum += count ? 1ull : fixed(v);
        }
        return meet(m, turn, blocks, rank, sum, Sum{});
      };
      unsigned long long need;
      if (rule == 0) {
        need = (unsigned long long)(target - c_front);  // whole numbers
      } else {
        const double missing = ceil((target - w_front) / unit) - (double)front_in_bin;
        need = missing < 1.0 ? 1ull : (unsigned long long)missing;
      }
      const unsigned long long most = amount(0, rule == 0);
      need = need < most ? need : most;
      const unsigned long long cut = cut_by_bits([&](unsigned long long c) { return amount(c, rule == 0); }, need);
      kept_sum = w_front + unit * (double)(front_in_bin + amount(cut, false));
      return cut;
    };
    unsigned long long cut = 0;
    if (k > 0 && (unsigned)k < left) cut = border(0, (double)k);
    if (p < 1.f) {
      const unsigned long long by_share = border(1, (double)p * kept_sum);
      cut = by_share > cut ? by_share : cut;
    }
    cut = cut < first ? cut : first;
    const float cut_value = cut == 0 ? -INFINITY : value_of(cut);
#pragma unroll 2
    for (int i0 = 0; i0 < padded; i0 += 4 * THREADS) {  // (whole warps)
      const int i = i0 + 4 * tid;
      const float4 f = i < padded ? four_at(i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (!__any_sync(0xffffffffu, fmaxf(fmaxf(f.x, f.y), fmaxf(f.z, f.w)) >= cut_value)) continue;
      const float v[4] = {f.x, f.y, f.z, f.w};
      unsigned random[4];
      bool tried[4], any = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        tried[j] = false;
        if (v[j] >= cut_value && (v[j] > cut_value || place_of(v[j], (unsigned)(lo + i + j)) >= cut)) {
          random[j] = random_of(of_step, (unsigned)(lo + i + j));
          any |= tried[j] = may_win(random[j], weight_of(v[j]));
        }
      }
      if (__any_sync(0xffffffffu, any)) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (tried[j]) try_token(v[j], random[j], (unsigned)(lo + i + j));
        share_the_best();
      }
    }
  }
  double log_all = 0.0;
  unsigned long long sum = (unsigned long long)__double_as_longlong(all);
  if (cuts) {
    meet_pair(m, turn, blocks, rank, best, Larger{}, (unsigned long long*)nullptr, SumDoubles{},
              [&] { if (tid == 0) log_all = log(all); });
  } else {
    meet_pair(m, turn, blocks, rank, best, Larger{}, &sum, SumDoubles{}, [] {});
    if (tid == 0) log_all = log(__longlong_as_double((long long)sum));
  }
  const int token = (int)(ID_MASK - (unsigned)(best & ID_MASK));
  if (tid == 0 && token >= lo && token < hi) {
    a.out[r] = token;
    if (a.also != nullptr) a.also[r] = token;
    // (in 64 bits, rounded once: what the sum's weights are off by is all that is left, below a rounding's size)
    a.logprobs[r] = (float)(((double)values[token - lo] - (double)M) / (greedy ? 1.0 : (double)T) - log_all);
  }
  // (the last meeting's barrier is behind every word to another block)
}

// How many clusters of 1, 2, 4, 8 and 16 blocks the device runs at once where an SM has one block (0: none),
// with the kernel set up for it.
int clusters_at_once(const int** counts) {
  static int of_device[64][6] = {};  // the last number: made
  int device = 0;
  cudaGetDevice(&device);
  if (device < 0 || device >= 64) device = 63;
  int* const of = of_device[device];
  if (of[5] == 0) {
    const int most = MAX_CHUNK * 4 + (int)sizeof(Bins);
    cudaError_t e = cudaSuccess;
    for (auto kernel : {sample_rules_kernel<1>, sample_rules_kernel<2>}) {
      if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
      if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    }
    if (e != cudaSuccess) return fb_fail(2, "sample_rules: setting the kernel up: %s", cudaGetErrorString(e));
    for (int i = 0; i < 5; ++i) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1, 1, 1 << i);
      cfg.blockDim = dim3(THREADS);
      cfg.dynamicSmemBytes = most;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1 << i;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, sample_rules_kernel<1>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
      }
      of[i] = n;
    }
    of[5] = 1;
  }
  *counts = of;
  return 0;
}

constexpr int TWO_AN_SM = 20000;  // logits a block at most for two of them on an SM

// Blocks a row. The most that leave every block an SM of its own (eight; sixteen for long rows), down to 1,000
// logits a block; where even the fewest that hold a row do not, the fewest of which two fit an SM. Measured with
// 1, 2, 4, 8, 16 blocks, plain draws and top-p:
//   1 row of 128,256: -, -, 15.9 and 22.7, 11.0 and 18.6, 8.2 and 15.5 us;
//   33 rows of 32,000: 16.0 and 43, 11.2 and 31, 8.7 and 22, 9.4 and 27, 19.5 and 52;
//   64 rows of 32,000: 16.2 and 43, 11.5 and 32, 11.8 and 30, 18.3 and 45, 35 and 84;
//   256 rows of 8,000: 12 and 30, 17 and 40, 28 and 63, 51 and 123, 115 and 286.
int blocks_a_row(int n, int V, int* blocks, int* an_sm) {
  const int* at_once;
  if (int rc = clusters_at_once(&at_once)) return rc;
  const bool wide = at_once[4] > 0;
  *an_sm = 1;
  if (wide && (V > 8 * MAX_CHUNK || (V >= 65536 && 16 * n <= sm_count()))) {
    *blocks = 16;
    if (n > at_once[4] && V <= 16 * TWO_AN_SM) *an_sm = 2;
    return 0;
  }
  for (int i = 3; i >= 0; --i) {
    if ((i > 0 && V < 1000 << i) || V > MAX_CHUNK << i) continue;
    if (n <= at_once[i]) {
      *blocks = 1 << i;
      return 0;
    }
  }
  *blocks = 1;
  while (*blocks < 8 && V > TWO_AN_SM * *blocks) *blocks *= 2;
  if (V <= TWO_AN_SM * *blocks) *an_sm = 2;
  return 0;
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
  if (n == 0) return 0;  // (its rows' arrays are empty too, and have no address)
  SampleArgs a{};
  a.edits = fb_unpack_edits(edits);
  if (int rc = fb_check_edits("sample_rules", a.edits, V)) return rc;
  FB_REQUIRE(record == nullptr || a.edits.counts != nullptr, "sample_rules: tokens to record, and no history");
  int blocks = 0, an_sm = 1;
  if (int rc = blocks_a_row(n, V, &blocks, &an_sm)) return rc;
  FB_REQUIRE(V <= blocks * MAX_CHUNK, "sample_rules: a vocabulary of %d (%d at most here)", V, blocks * MAX_CHUNK);
  a.logits = logits; a.row_stride = row_stride; a.V = V;
  a.chunk = ((V + blocks - 1) / blocks + 31) / 32 * 32;  // whole words of the bits
  a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p;
  a.streams = streams; a.steps = steps; a.record = record;
  a.out = out; a.logprobs = logprobs; a.also = also;
  fb_launch_cluster(an_sm == 2 ? sample_rules_kernel<2> : sample_rules_kernel<1>, dim3(n, 1, blocks), dim3(THREADS),
                    (size_t)a.chunk * 4 + sizeof(Bins), stream,
                    (unsigned)blocks, a);
  return fb_check_launch("sample_rules");
}
