// What a request's own edits do to a logit, for the kernels that write edited logits
// (logit_edits.cu) and that draw from them (sample_rules.cu).
//
//   seen in the history (prompt or generated):  v = v > 0 ? v / repetition : v * repetition
//   generated c > 0 times:                      v = (v - frequency * c) - presence
//   then                                        v = v + bias
//   not allowed:                                v = -inf, whatever v was
//
// Every operation is rounded by itself (no fused multiply-add), so that an edited logit, and with it
// every border that a rule draws between two of them, is one 32-bit number whoever computes it.
#pragma once

#include "common.cuh"

constexpr int FB_IN_PROMPT = 1 << 30;  // bit 30 of a history's word; bits 0..29 count

// Tables and per-row parameters on the device; null where a step has none of a kind.
struct FbLogitEdits {
  int* counts;               // [history_rows_in_table, V]
  unsigned* seen;            // [.., seen_words]: a bit a token, set where its count is not 0
  const int* history_row;    // [n]: a row's history, outside of the table: none
  int history_rows, seen_words;
  const float* repetition;   // [n] each
  const float* frequency;
  const float* presence;
  const int* bias_starts;    // [n + 1]
  const int* bias_ids;       // ascending within a row
  const float* bias_values;
  int bias_total;
  const unsigned* allowed;   // [masks, seen_words]
  const int* allowed_row;    // [n]: a row's mask, outside of the table: none
  int masks;
};

// The edits of one row.
struct FbRowEdits {
  int* counts;
  unsigned* seen;
  const unsigned* allowed;
  float repetition, frequency, presence;
  int bias_from, bias_to;
};

__device__ __forceinline__ FbRowEdits fb_row_edits(const FbLogitEdits& e, int r, int V) {
  FbRowEdits row{nullptr, nullptr, nullptr, 1.f, 0.f, 0.f, 0, 0};
  if (e.counts != nullptr) {
    const int h = e.history_row[r];
    if (h >= 0 && h < e.history_rows) {
      row.counts = e.counts + (size_t)h * V;
      row.seen = e.seen + (size_t)h * e.seen_words;
      if (e.repetition != nullptr) row.repetition = e.repetition[r];
      if (e.frequency != nullptr) row.frequency = e.frequency[r];
      if (e.presence != nullptr) row.presence = e.presence[r];
    }
  }
  if (e.bias_starts != nullptr) {
    row.bias_from = max(0, e.bias_starts[r]);
    row.bias_to = min(e.bias_total, e.bias_starts[r + 1]);
  }
  if (e.allowed != nullptr) {
    const int m = e.allowed_row[r];
    if (m >= 0 && m < e.masks) row.allowed = e.allowed + (size_t)m * e.seen_words;
  }
  return row;
}

// The penalties on a token whose bit in `seen` is set; `word` is its word of the history.
__device__ __forceinline__ float fb_penalised(const FbRowEdits& e, float v, int word) {
  v = v > 0.f ? __fdiv_rn(v, e.repetition) : __fmul_rn(v, e.repetition);
  const int said = word & (FB_IN_PROMPT - 1);
  if (said > 0) v = __fsub_rn(__fsub_rn(v, __fmul_rn(e.frequency, (float)said)), e.presence);
  return v;
}

// The biases of a row that fall into [lo, hi), added to the values of allowed tokens, which lie from lo
// on. Threads look at the row's whole list side by side (a request has some hundreds at most). Equal
// ids stand side by side, and the first one's thread adds them all, in order.
__device__ __forceinline__ void fb_add_biases(const FbLogitEdits& e, const FbRowEdits& row, float* values,
                                              int lo, int hi) {
  for (int i = row.bias_from + (int)threadIdx.x; i < row.bias_to; i += (int)blockDim.x) {
    const int id = e.bias_ids[i];
    if (id < lo || id >= hi || (i > row.bias_from && e.bias_ids[i - 1] == id)) continue;
    if (row.allowed != nullptr && !(row.allowed[id >> 5] >> (id & 31) & 1u)) continue;
    float v = values[id - lo];
    for (int j = i; j < row.bias_to && e.bias_ids[j] == id; ++j) v = __fadd_rn(v, e.bias_values[j]);
    values[id - lo] = v;
  }
}

// `packed` (on the host): the 15 fields in their order, as the Python side lays them down; null: none.
inline FbLogitEdits fb_unpack_edits(const long long* packed) {
  FbLogitEdits e{};
  if (packed == nullptr) return e;
  e.counts = (int*)packed[0];
  e.seen = (unsigned*)packed[1];
  e.history_row = (const int*)packed[2];
  e.history_rows = (int)packed[3];
  e.seen_words = (int)packed[4];
  e.repetition = (const float*)packed[5];
  e.frequency = (const float*)packed[6];
  e.presence = (const float*)packed[7];
  e.bias_starts = (const int*)packed[8];
  e.bias_ids = (const int*)packed[9];
  e.bias_values = (const float*)packed[10];
  e.bias_total = (int)packed[11];
  e.allowed = (const unsigned*)packed[12];
  e.allowed_row = (const int*)packed[13];
  e.masks = (int)packed[14];
  return e;
}

inline int fb_check_edits(const char* what, const FbLogitEdits& e, int V) {
  const bool words = e.counts == nullptr && e.allowed == nullptr;
  FB_REQUIRE(words || e.seen_words >= (V + 31) / 32, "%s: rows of %d bit words for %d tokens", what,
             e.seen_words, V);
  FB_REQUIRE(e.counts == nullptr || (e.seen && e.history_row && e.history_rows > 0),
             "%s: a history needs its counts, its bits and the rows' places", what);
  FB_REQUIRE(e.allowed == nullptr || (e.allowed_row && e.masks > 0), "%s: masks need the rows' places", what);
  FB_REQUIRE(e.bias_starts == nullptr || (e.bias_total >= 0 && (e.bias_total == 0 || (e.bias_ids && e.bias_values))),
             "%s: biases need their ids and values", what);
  return 0;
}
