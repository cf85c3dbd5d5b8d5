// Edited logits, and the histories that the penalties look at.
//
// A history is a row of a table: `counts` has a word a token (how often it was generated, and bit 30
// if the prompt holds it), `seen` a bit a token. The edits read the bits of all tokens and the words
// of those alone whose bit is set: an eighth of a byte a token instead of four.
#include "logit_edits.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int EACH = 16;                // logits of a thread
constexpr int TILE = THREADS * EACH;    // and of a block
constexpr int WARP_TILE = 32 * EACH;

// Bit j of lane l: bit l of word j of 16 side by side (those past `end` count as zeros). One load of a
// lane each and an exchange, where a word for all lanes would be a load for every 32 tokens.
__device__ __forceinline__ unsigned bits_of(const unsigned* words, int end, int lane) {
  const unsigned mine = lane < EACH && lane < end ? words[lane] : 0u;
  unsigned bits = 0u;
#pragma unroll
  for (int j = 0; j < EACH; ++j) bits |= (__shfl_sync(0xffffffffu, mine, j) >> lane & 1u) << j;
  return bits;
}

// Block (c, r) edits logits [c * TILE, ..) of row r; a warp has 512 side by side, so that it reads whole lines
// whatever a row's start is aligned to, and a thread 16, all asked for together. They go out as they are, or as
// -inf, as soon as they are there. The few tokens that the history holds are put on a list meanwhile, and the
// block's threads then work it off in `out`, one load of a count each, all at once; biases follow. 64 rows of
// 128,256 with 4,000 tokens, 300 biases and masks: 18.0 us from memory, 68 MB at 3.8 TB/s (13.5 from L2); what is
// left to the copy rate's 10.4 are chains of three loads in two rounds of blocks. (From L2: six blocks an SM instead of eight 14.6, 8 logits a thread
// 15.5, the tile in shared memory until its edits are done 16.6; where each thread looked after its own tokens
// the counts came one after another, and a warp went through the penalties for every 32 tokens of which it
// held one: 31.)
__global__ void __launch_bounds__(THREADS, 8)
edit_logits_kernel(const float* logits, long long row_stride, int V, float* out, long long out_stride,
                   const FbLogitEdits edits) {
  fb_pdl_wait();
  __shared__ unsigned short hits[TILE];
  __shared__ int hit_count;
  const int r = blockIdx.y, lo = blockIdx.x * TILE, hi = min(V, lo + TILE), tid = threadIdx.x;
  const int lane = tid & 31, first = (tid >> 5) * WARP_TILE + lane;  // in the tile; the next one is 32 further
  const float* from = logits + (size_t)r * row_stride + lo;
  float* to = out + (size_t)r * out_stride + lo;
  const int here = hi - lo;
  float v[EACH];
#pragma unroll
  for (int j = 0; j < EACH; ++j) v[j] = first + 32 * j < here ? from[first + 32 * j] : 0.f;
  const FbRowEdits row = fb_row_edits(edits, r, V);
  const int word0 = (lo + first - lane) >> 5, words = ((V + 31) >> 5) - word0;
  const unsigned ok = row.allowed != nullptr ? bits_of(row.allowed + word0, words, lane) : ~0u;
  const unsigned held = row.counts != nullptr ? bits_of(row.seen + word0, words, lane) & ok : 0u;
  if (row.counts != nullptr) {  // (the whole block)
    if (tid == 0) hit_count = 0;
    __syncthreads();
    // the places of this warp's tokens on the list
    const int mine = __popc(held);
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
    int at = 0;
    if (lane == 31 && upto > 0) at = atomicAdd(&hit_count, upto);
    at = __shfl_sync(0xffffffffu, at, 31) + upto - mine;
    for (unsigned left = held; left != 0u; left &= left - 1)
      hits[at++] = (unsigned short)(first + 32 * (__ffs(left) - 1));
  }
#pragma unroll
  for (int j = 0; j < EACH; ++j)
    if (first + 32 * j < here) to[first + 32 * j] = (ok >> j & 1u) ? v[j] : -INFINITY;
  if (row.counts != nullptr) {
    __syncthreads();  // the list, and what the block's threads wrote
    for (int i = tid; i < hit_count; i += THREADS) {
      const int where = hits[i];
      if (where < here) to[where] = fb_penalised(row, to[where], row.counts[lo + where]);
    }
  }
  if (row.bias_from < row.bias_to) {
    __syncthreads();
    fb_add_biases(edits, row, to, lo, hi);
  }
}

// Token i goes into history rows[i] (outside of the table: skipped, like a token outside of the
// vocabulary). what 0: the prompt holds it; 1: it was generated once more; 2: once less. Integer
// atomics: the same table whatever the order, and however often a token comes in one call.
__global__ void record_tokens_kernel(int* counts, unsigned* seen, int history_rows, int seen_words, int V,
                                     const int* rows, const int* tokens, int n, int what) {
  fb_pdl_wait();
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) {
    const int h = rows[i], t = tokens[i];
    if (h < 0 || h >= history_rows || t < 0 || t >= V) continue;
    int* word = counts + (size_t)h * V + t;
    unsigned* bits = seen + (size_t)h * seen_words + (t >> 5);
    const unsigned bit = 1u << (t & 31);
    if (what == 0) {
      atomicOr(word, FB_IN_PROMPT);
      atomicOr(bits, bit);
    } else if (what == 1) {
      atomicAdd(word, 1);
      atomicOr(bits, bit);
    } else {
      int held = *(volatile int*)word;  // down to zero and no further
      while ((held & (FB_IN_PROMPT - 1)) > 0) {
        const int before = atomicCAS(word, held, held - 1);
        if (before == held) {
          if (held == 1) atomicAnd(bits, ~bit);
          break;
        }
        held = before;
      }
    }
  }
}
}  // namespace

// out[r, i] = the edited logits[r, i] (see logit_edits.cuh), float32; `out` may be `logits`.
// `edits`: on the host, the fields of FbLogitEdits as 64-bit integers.
FB_API int fb_edit_logits(const float* logits, long long row_stride, int n, int V, float* out,
                          long long out_stride, const long long* edits, cudaStream_t stream) {
  FB_REQUIRE(n >= 0 && V > 0 && row_stride >= V && out_stride >= V, "edit_logits: bad sizes n=%d V=%d", n, V);
  FB_REQUIRE(n <= 65535, "edit_logits: %d rows (65535 at most)", n);
  if (n == 0) return 0;  // (its rows' arrays are empty too, and have no address)
  const FbLogitEdits e = fb_unpack_edits(edits);
  if (int rc = fb_check_edits("edit_logits", e, V)) return rc;
  fb_launch(edit_logits_kernel, dim3((V + TILE - 1) / TILE, n), dim3(THREADS), 0, stream, logits,
            row_stride, V, out, out_stride, e);
  return fb_check_launch("edit_logits");
}

FB_API int fb_record_tokens(int* counts, unsigned* seen, int history_rows, int seen_words, int V,
                            const int* rows, const int* tokens, int n, int what, cudaStream_t stream) {
  FB_REQUIRE(n >= 0 && V > 0 && history_rows > 0 && seen_words >= (V + 31) / 32,
             "record_tokens: bad sizes n=%d V=%d", n, V);
  FB_REQUIRE(what >= 0 && what <= 2, "record_tokens: what=%d", what);
  if (n == 0) return 0;
  fb_launch(record_tokens_kernel, dim3((n + 255) / 256 < 1024 ? (n + 255) / 256 : 1024), dim3(256), 0,
            stream, counts, seen, history_rows, seen_words, V, rows, tokens, n, what);
  return fb_check_launch("record_tokens");
}
