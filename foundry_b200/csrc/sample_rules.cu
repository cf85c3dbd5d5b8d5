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
constexpr int MAX_CHUNK = 46080;  // a block's logits in shared memory: 180 KB, beside 42 KB of bins
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

// The upper half of token i's random number; its top 24 bits are those of the number that sampling.cu
// makes (whose last exclusive-or does not reach them).
__device__ __forceinline__ unsigned random_of(unsigned long long of_step, unsigned i) {
  unsigned long long z = of_step + GOLDEN * ((unsigned long long)i + 1);
  z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ULL;
  return (unsigned)(((z ^ (z >> 27)) * 0x94d049bb133111ebULL) >> 32);
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

// Tokens by their distance d = (M - v) / T from the best one: bins of 1 / 64, the last one for all
// that is further. Inside a bin the weights exp(-d) are exp(-b / 64) (1 - part), with part below
// 1 / 64; its 22-bit fraction adds up as whole numbers, so that the sums do not depend on the order
// in which threads come. What the last bin weighs (V exp(-32) at most) is left out of the sums.
constexpr int BINS = 2048;
constexpr float BINS_PER_UNIT = 64.f;
constexpr int PART_BITS = 22;
constexpr int LISTED = 1024;  // tokens of a border's bin that are put in order in shared memory

// A distance in 64ths: its bin (an edge belongs to either side, always the same one), and 1 - exp(-x) of
// what is left of it, x <= 1 / 64, by its series (the next term is below 2^-28), in units of 2^-22. Whole
// numbers are made and taken off by adding 1.5 * 2^23, which leaves them in the last bits.
constexpr float TO_WHOLE = 12582912.f;
__device__ __forceinline__ bool in_last_bin(float t) { return !(t < (float)(BINS - 1)); }
__device__ __forceinline__ int bin_of(float t) {
  return in_last_bin(t) ? BINS - 1 : __float_as_int((t - 0.5f) + TO_WHOLE) & 0xffff;
}
__device__ __forceinline__ unsigned part_of(float t) {  // of a token in front of the last bin
  const float x = t - (((t - 0.5f) + TO_WHOLE) - TO_WHOLE);  // exact
  const float part = x * (65536.f - x * (512.f - x * (1024.f / 384.f)));
  return (unsigned)__float_as_int(part + TO_WHOLE) & 0x3ffffu;
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
  unsigned long long listed[LISTED];
  unsigned long long scan_warps[2][THREADS / 32];
  unsigned counted;
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

// A row by a cluster of `gridDim.z` blocks, each with `chunk` of its logits in shared memory.
__global__ void __launch_bounds__(THREADS)
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
  const float T = a.temperature != nullptr ? a.temperature[r] : 0.f;
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
  float top = -INFINITY;  // the thread's best value, and where it comes first
  int top_at = -1;
  // a value on its way out of the edits: NaN has no chance, like a token that is not allowed
  auto settle = [&](float v, int i, unsigned ok) {
    v = ok ? fmaxf(v, -INFINITY) : -INFINITY;
    if (v > top) { top = v; top_at = i; }
    return v;
  };
  auto come_in = [&](float v, int i, unsigned held, unsigned ok) {
    if (held & 1u) v = fb_penalised(row, v, row.counts[lo + i]);
    return biased ? v : settle(v, i, ok & 1u);
  };
  const unsigned* seen = row.counts != nullptr ? row.seen + (lo >> 5) : nullptr;
  const unsigned* allowed = row.allowed != nullptr ? row.allowed + (lo >> 5) : nullptr;
  int done = 0;
  if ((reinterpret_cast<uintptr_t>(from) & 15) == 0) {
    done = mine & ~3;
    constexpr int AHEAD = 4;
    for (int i0 = tid * 4; i0 < done; i0 += THREADS * 4 * AHEAD) {
      float4 got[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int i = i0 + j * THREADS * 4;
        if (i < done) got[j] = *reinterpret_cast<const float4*>(from + i);
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int i = i0 + j * THREADS * 4;
        if (i >= done) break;
        const unsigned held = seen != nullptr ? seen[i >> 5] >> (i & 31) : 0u;
        const unsigned ok = allowed != nullptr ? allowed[i >> 5] >> (i & 31) : ~0u;
        got[j].x = come_in(got[j].x, i, held, ok);
        got[j].y = come_in(got[j].y, i + 1, held >> 1, ok >> 1);
        got[j].z = come_in(got[j].z, i + 2, held >> 2, ok >> 2);
        got[j].w = come_in(got[j].w, i + 3, held >> 3, ok >> 3);
        *reinterpret_cast<float4*>(values + i) = got[j];
      }
    }
  }
  for (int i = done + tid; i < mine; i += THREADS) {
    const unsigned held = seen != nullptr ? seen[i >> 5] >> (i & 31) : 0u;
    const unsigned ok = allowed != nullptr ? allowed[i >> 5] >> (i & 31) : ~0u;
    values[i] = come_in(from[i], i, held, ok);
  }
  if (cuts)
    for (int b = tid; b < BINS; b += THREADS) bins.count[b] = bins.part[b] = 0;
  __syncthreads();
  if (biased) {
    fb_add_biases(a.edits, row, values, lo, hi);
    __syncthreads();
    for (int i = tid; i < mine; i += THREADS)
      values[i] = settle(values[i], i, allowed != nullptr ? allowed[i >> 5] >> (i & 31) & 1u : 1u);
  }
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
  const float inv_t = greedy ? 1.f : 1.0f / T;
  // exp(-(M - v) / T) as a power of two, its factor rounded once from 64 bits
  const float log2_t = (float)(-1.4426950408889634 / (greedy ? 1.0 : (double)T));
  auto weight_of = [&](float v) { return exp2_fast((M - v) * log2_t); };
  auto distance = [&](float v) { return (M - v) * inv_t; };
  const float bins_t = inv_t * BINS_PER_UNIT;
  auto binned = [&](float v) { return (M - v) * bins_t; };
  const unsigned long long stream = a.streams != nullptr ? (unsigned long long)a.streams[r] : 0ULL;
  const unsigned long long step = a.steps != nullptr ? (unsigned long long)a.steps[r] : 0ULL;
  const unsigned long long of_step = mix64(stream + GOLDEN * (step + 1));
  // The winner of the draw so far, as a place of its score. A token of weight w beats score s where
  // -log u < w exp(-s), and -log u >= 1 - u: all but a few of the tokens need no logarithm (with a
  // thousandth more of the right side than rounding could ask for; 1 - u from 23 of its bits, a unit
  // less). The first token's score is where every thread starts: that one is always kept.
  const unsigned first_id = ID_MASK - (unsigned)(first & ID_MASK);
  unsigned long long best = greedy ? first : place_of(gumbel(random_of(of_step, first_id)), first_id);
  float beaten = greedy ? 0.f : 1.001f * expf(-value_of(best));
  auto try_token = [&](float v, float w, unsigned id) {
    const unsigned random = random_of(of_step, id);
    if ((2.0f - 0x1p-22f) - __uint_as_float(random >> 9 | 0x3f800000u) > w * beaten) return;
    const unsigned long long score = place_of(gumbel(random) - distance(v), id);
    if (score > best) {
      best = score;
      beaten = 1.001f * expf(-value_of(best));
    }
  };
  double all = 0.0;
  if (!cuts) {  // one pass: the sum of the weights and the draw
    if (greedy) {
#pragma unroll 4
      for (int i = tid; i < mine; i += THREADS) all += (double)weight_of(values[i]);
    } else {
#pragma unroll 4
      for (int i = tid; i < mine; i += THREADS) {
        const float v = values[i], w = weight_of(v);
        all += (double)w;
        if (w >= least && v != -INFINITY) try_token(v, w, (unsigned)(lo + i));
      }
    }
    all = __longlong_as_double((long long)meet(m, turn, blocks, rank,
                                               (unsigned long long)__double_as_longlong(all), SumDoubles{}));
  } else {
#pragma unroll 4
    for (int i = tid; i < mine; i += THREADS) {
      const float v = values[i], t = binned(v);
      if (!in_last_bin(t)) {
        const int b = bin_of(t);
        atomicAdd(&bins.count[b], 1u);
        atomicAdd(&bins.part[b], part_of(t));
      } else if (v != -INFINITY) {  // it may hold nearly all tokens: their number is made by warps
        const unsigned together = __activemask();
        if ((tid & 31) == __ffs(together) - 1) atomicAdd(&bins.count[BINS - 1], __popc(together));
      }
    }
    cluster_sync();
    // each block adds up its share of the bins over the cluster and tells everybody
    const int share = BINS / blocks;
    for (int i = tid; i < share; i += THREADS) {
      const int b = (int)rank * share + i;
      unsigned count = 0;
      unsigned long long part = 0;
      for (int o = 0; o < blocks; ++o) {
        count += load_at(&bins.count[b], o);
        part += load_at(&bins.part[b], o);
      }
      const double size = (double)(((unsigned long long)count << PART_BITS) - part) * (1.0 / (1 << PART_BITS));
      const float weight = b == BINS - 1 ? 0.f : (float)(exp(-(double)b / BINS_PER_UNIT) * size);
      for (int o = 0; o < blocks; ++o) {
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
      for (int o = 0; o < THREADS / 32; ++o) {
        const double ow = __longlong_as_double((long long)bins.scan_warps[1][o]);
        if (o < (tid >> 5)) {
          front_c += (unsigned)bins.scan_warps[0][o];
          front_w += ow;
        }
        left += (unsigned)bins.scan_warps[0][o];
        all += ow;
      }
      count_before = front_c + upto_c - c;
      weight_before = front_w + (upto_w - w);
    }
    // The border of a rule: the last bin with tokens whose front is below `target`, put in order, and
    // of its tokens the last one whose front is. `by_count`: fronts count tokens, else they weigh.
    double front_sum = 0.0;  // what the last border keeps weighs
    bool listed_before = false;
    auto border = [&](bool by_count, double target) -> unsigned long long {
      unsigned long long at = 0;  // (bin + 1, what stands in front of it: a thread of the block knows)
      {
        unsigned c = count_before;
        double w = weight_before;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
          if (counts[j] != 0 && (by_count ? (double)c : w) < target) at = (unsigned long long)(tid * EACH + j + 1);
          c += counts[j];
          w += (double)weights[j];
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, at, o);
        at = other > at ? other : at;
      }
      __syncthreads();
      if ((tid & 31) == 0) bins.scan_warps[0][tid >> 5] = at;
      if (tid == 0) bins.counted = 0;
      __syncthreads();
      for (int o = 0; o < THREADS / 32; ++o) at = bins.scan_warps[0][o] > at ? bins.scan_warps[0][o] : at;
      if (at == 0) {  // a share of nothing
        front_sum = 1.0;
        return first;
      }
      const int b = (int)at - 1;
      // the owner of that bin tells what stands in front of it
      __syncthreads();
      if (tid == b / EACH) {
        unsigned c = count_before;
        double w = weight_before;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
          if (j < b % EACH) { c += counts[j]; w += (double)weights[j]; }
        }
        bins.scan_warps[0][0] = c;
        bins.scan_warps[1][0] = (unsigned long long)__double_as_longlong(w);
      }
      __syncthreads();
      const double c_front = (double)bins.scan_warps[0][0];
      const double w_front = __longlong_as_double((long long)bins.scan_warps[1][0]);
      const double unit = b == BINS - 1 ? 0.0 : exp(-(double)b / BINS_PER_UNIT) * (1.0 / (1 << PART_BITS));
      const unsigned n = bins.all_count[b];
      auto fixed = [&](float v) { return (unsigned long long)weight_in_bin(binned(v)); };
      if (n <= LISTED) {
        // everybody gets everybody's tokens of the bin; a block's stand behind those of lower ranks
        if (listed_before) cluster_sync();  // everybody is through with the list of the border before
        listed_before = true;
        unsigned base = 0;
        for (int o = 0; o < (int)rank; ++o) base += load_at(&bins.count[b], o);
        for (int i = tid; i < mine; i += THREADS) {
          const float v = values[i];
          if (v == -INFINITY || bin_of(binned(v)) != b) continue;
          const unsigned slot = base + atomicAdd(&bins.counted, 1u);
          const unsigned long long place = place_of(v, (unsigned)(lo + i));
          for (int o = 0; o < blocks; ++o) store_at(&bins.listed[slot], o, place);
        }
        cluster_sync();
        // in order, the first place first (a bitonic network; zeros behind the tokens)
        unsigned padded = 32;
        while (padded < n) padded *= 2;
        for (unsigned i = n + tid; i < padded; i += THREADS) bins.listed[i] = 0;
        __syncthreads();
        for (unsigned size = 2; size <= padded; size *= 2) {
          for (unsigned stride = size / 2; stride > 0; stride /= 2) {
            if ((unsigned)tid < padded / 2) {
              const unsigned i = 2 * tid - (tid & (stride - 1)), j = i + stride;
              const unsigned long long x = bins.listed[i], y = bins.listed[j];
              if ((x < y) == ((i & size) == 0)) { bins.listed[i] = y; bins.listed[j] = x; }
            }
            __syncthreads();
          }
        }
        // a thread has two of them side by side: what stands in front of each, and is it kept
        unsigned long long weighs[2], upto;
#pragma unroll
        for (int j = 0; j < 2; ++j) weighs[j] = 2u * tid + j < n ? fixed(value_of(bins.listed[2 * tid + j])) : 0ull;
        upto = weighs[0] + weighs[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned long long other = __shfl_up_sync(0xffffffffu, upto, o);
          if ((tid & 31) >= o) upto += other;
        }
        if ((tid & 31) == 31) bins.scan_warps[1][tid >> 5] = upto;
        __syncthreads();
        unsigned long long in_front = upto - weighs[0] - weighs[1];
        for (int o = 0; o < (tid >> 5); ++o) in_front += bins.scan_warps[1][o];
        unsigned long long kept = 0, many = 0;  // what the kept ones weigh, and how many they are
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const unsigned i = 2 * tid + j;
          if (i < n && (by_count ? c_front + (double)i : w_front + unit * (double)in_front) < target) {
            kept = in_front + weighs[j];
            many = i + 1;
          }
          in_front += weighs[j];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {  // both grow along the list
          const unsigned long long k2 = __shfl_xor_sync(0xffffffffu, kept, o);
          const unsigned long long m2 = __shfl_xor_sync(0xffffffffu, many, o);
          kept = k2 > kept ? k2 : kept;
          many = m2 > many ? m2 : many;
        }
        __syncthreads();
        if ((tid & 31) == 0) {
          bins.scan_warps[0][tid >> 5] = many;
          bins.scan_warps[1][tid >> 5] = kept;
        }
        __syncthreads();
        for (int o = 0; o < THREADS / 32; ++o) {
          many = bins.scan_warps[0][o] > many ? bins.scan_warps[0][o] : many;
          kept = bins.scan_warps[1][o] > kept ? bins.scan_warps[1][o] : kept;
        }
        const unsigned long long last = bins.listed[many > 0 ? many - 1 : 0];
        __syncthreads();
        front_sum = w_front + unit * (double)kept;
        return last;
      }
      auto amount = [&](unsigned long long cut, bool count) {
        unsigned long long sum = 0;
        for (int i = tid; i < mine; i += THREADS) {
          const float v = values[i];
          if (v == -INFINITY || place_of(v, (unsigned)(lo + i)) < cut || bin_of(binned(v)) != b) continue;
          sum += count ? 1ull : fixed(v);
        }
        return meet(m, turn, blocks, rank, sum, Sum{});
      };
      unsigned long long need;
      if (by_count) {
        need = (unsigned long long)(target - c_front);  // whole numbers
      } else {
        const double missing = ceil((target - w_front) / unit);
        need = missing < 1.0 ? 1ull : (unsigned long long)missing;
      }
      const unsigned long long most = amount(0, by_count);
      need = need < most ? need : most;
      const unsigned long long cut = cut_by_bits([&](unsigned long long c) { return amount(c, by_count); }, need);
      front_sum = w_front + unit * (double)amount(cut, false);
      return cut;
    };
    unsigned long long cut = 0;
    double kept_sum = all;
    if (k > 0 && (unsigned)k < left) {
      cut = border(true, (double)k);
      kept_sum = front_sum;
    }
    if (p < 1.f) {
      const unsigned long long by_share = border(false, (double)p * kept_sum);
      cut = by_share > cut ? by_share : cut;
    }
    cut = cut < first ? cut : first;
    const float cut_value = cut == 0 ? -INFINITY : value_of(cut);
#pragma unroll 4
    for (int i = tid; i < mine; i += THREADS) {
      const float v = values[i];
      if (v < cut_value || v == -INFINITY) continue;
      if (v == cut_value && place_of(v, (unsigned)(lo + i)) < cut) continue;
      const float w = weight_of(v);
      if (w >= least) try_token(v, w, (unsigned)(lo + i));
    }
  }
  if (!greedy) best = meet(m, turn, blocks, rank, best, Larger{});
  const int token = (int)(ID_MASK - (unsigned)(best & ID_MASK));
  if (tid == 0 && token >= lo && token < hi) {
    a.out[r] = token;
    if (a.also != nullptr) a.also[r] = token;
    a.logprobs[r] = (float)(-(double)distance(values[token - lo]) - log(all));
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
                                         MAX_CHUNK * 4 + (int)sizeof(Bins));
    if (e != cudaSuccess) return fb_fail(2, "sample_rules: shared memory opt-in: %s", cudaGetErrorString(e));
  }
  fb_launch_cluster(sample_rules_kernel, dim3(n, 1, blocks), dim3(THREADS),
                    (size_t)a.chunk * 4 + sizeof(Bins), stream,
                    (unsigned)blocks, a);
  return fb_check_launch("sample_rules");
}
