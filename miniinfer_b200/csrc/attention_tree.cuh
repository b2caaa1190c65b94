// What the kernels of attention over a tree of new tokens share: their arguments, which keys a row sees, and the pieces' merge.
//
// An item (a request) has `start` = ctx_len - q_len context keys and q_len new tokens, whose keys and values lie behind them in its pages:
// token t's at place start + t, whatever its position is.  A token sees the context keys, those further than `window` positions back excepted,
// and of the new ones those whose bit is set in its mask (a node's ancestors and itself).  A key's position is its place for the context and
// positions[] for the new tokens - one of start .. ctx_len - 1.
//
// Query rows of one item and key/value head lie behind one another, [token, head of the group]: row = token * G + g.
#pragma once

#include "attention_scores.cuh"
#include "common.cuh"

namespace mi_tree {

struct Args {
  void* out;                     // [T, nh * hd]
  const void* qkv;               // [T, width]: the queries are the first nh * hd values of a row
  const void* kv;                // [pages, 2, nkv, page_size, hd]
  const int* block_table; int bt_stride;
  const int *q_start, *q_len, *ctx_len, *seq_slot;      // [items]
  const int* mask; int words;    // [T, words]: bit j of a token's row - it sees new token j of its item
  const int* positions;          // [T]; read with a window only
  const float* sink;             // [nh] or null
  float *part_o, *part_ml;       // sums of pieces that are not normalised: [.., hd], and base-2 maximum and sum
  int items, T, width, nh, nkv, G, hd, pages, page_size, window, max_q;
  float scale, softcap;
};

// One item as the kernels walk it; sizes that make no sense are cut to ones that stay in bounds.
struct Item {
  int row0, n, start, ctx;       // first token, tokens, context keys, all keys
  const int* bt;
};
__device__ __forceinline__ Item item_of(const Args& a, int b) {
  Item it;
  it.row0 = max(a.q_start[b], 0);
  it.ctx = (int)max(0ll, min((long long)a.ctx_len[b], (long long)a.bt_stride * a.page_size));
  it.n = min(min(a.q_len[b], a.max_q), min(it.ctx, a.T - it.row0));
  it.n = max(it.n, 0);
  it.start = it.ctx - it.n;
  it.bt = a.block_table + (size_t)a.seq_slot[b] * a.bt_stride;
  return it;
}
__device__ __forceinline__ int page_of(const Args& a, const Item& it, int key) {
  return min(max(it.bt[min(key / a.page_size, a.bt_stride - 1)], 0), a.pages - 1);
}
// Keys from here on are visible to a token at position p, as far as the window goes.
__device__ __forceinline__ int window_begin(const Args& a, int p) { return a.window > 0 ? max(0, p - a.window + 1) : 0; }

// A score in base 2, as the online softmax takes it, exact to float32: the path whose inputs are float32.
__device__ __forceinline__ float logit2_exact(float raw, float scale, float softcap) {
  float x = raw * scale;
  if (softcap > 0.f) x = softcap * tanhf(x / softcap);
  return x * 1.4426950408889634f;
}

}  // namespace mi_tree
