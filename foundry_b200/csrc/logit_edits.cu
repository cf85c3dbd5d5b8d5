// Edited logits, and the histories that the penalties look at.
//
// A history is a row of a table: `counts` has a word a token (how often it was generated, and bit 30
// if the prompt holds it), `seen` a bit a token. The edits read the bits of all tokens and the words
// of those alone whose bit is set: an eighth of a byte a token instead of four.
#include "logit_edits.cuh"

namespace {

constexpr int TILE = 4096;     // logits a block edits
constexpr int THREADS = 256;

// Block (c, r) edits logits [c * TILE, ..) of row r: penalties as the logits come in, biases in shared
// memory, the mask as they go out.
__global__ void __launch_bounds__(THREADS)
edit_logits_kernel(const float* logits, long long row_stride, int V, float* out, long long out_stride,
                   const FbLogitEdits edits) {
  fb_pdl_wait();
  __shared__ float tile[TILE];
  const int r = blockIdx.y, lo = blockIdx.x * TILE, hi = min(V, lo + TILE);
  const float* from = logits + (size_t)r * row_stride;
  float* to = out + (size_t)r * out_stride;
  const FbRowEdits row = fb_row_edits(edits, r, V);
  for (int i = lo + threadIdx.x; i < hi; i += THREADS) {
    float v = from[i];
    if (row.counts != nullptr && (row.seen[i >> 5] >> (i & 31) & 1u)) v = fb_penalised(row, v, row.counts[i]);
    tile[i - lo] = v;
  }
  __syncthreads();
  fb_add_biases(edits, row, tile, lo, hi);
  __syncthreads();
  for (int i = lo + threadIdx.x; i < hi; i += THREADS) {
    const bool allowed = row.allowed == nullptr || (row.allowed[i >> 5] >> (i & 31) & 1u);
    to[i] = allowed ? tile[i - lo] : -INFINITY;
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
  const FbLogitEdits e = fb_unpack_edits(edits);
  if (int rc = fb_check_edits("edit_logits", e, V)) return rc;
  if (n == 0) return 0;
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
