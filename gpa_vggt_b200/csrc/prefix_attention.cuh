// What the kernels of the attention over a shared prefix have in common: the
// call's parameters, the rows of a tile and the partial outputs of key chunks.
#pragma once

#include "common.cuh"
#include "capi_util.h"

namespace gpa {
namespace prefix {

struct Params {
  const __nv_bfloat16 *q, *kp, *vp, *ko, *vo;
  const float* bias;
  const int32_t *own_len, *q_len;
  int requests, queries, heads, kv_heads, group, prefix, cache;
  int64_t q_sr, q_sh, q_sm, kp_sh, kp_sn, vp_sh, vp_sn, ko_sr, ko_sh, ko_sn, vo_sr, vo_sh, vo_sn, bias_sh;
  float scale, scale_log2;
  int causal;
  __nv_bfloat16* o;
  int64_t o_sr, o_sh, o_sm;
  float* lse;
  int64_t lse_sr, lse_sh;
  // rows_kernel's items: row tiles x chunks of the prefix per key head, then of each request's cache
  int rt1, s1, rt2, s2, chunk;   // chunk in keys; s1 + s2 partial outputs per row
  int64_t rows;                  // requests * queries * heads
  float* ws_o;                   // [s1 + s2][rows][D]
  float2* ws_ml;                 // [s1 + s2][rows]: maximum (log2 units) and sum
  // tc_kernel's: a row tile's outputs lie feature group by feature group, so that
  // its threads, one per row, write and read whole lines
  float4* tc_o;                  // [part_tiles(tc)][D / 4][128 rows], see part_tile
  float2* tc_ml;                 // [slots][blocks][128 rows]
  int32_t* tc_first;             // [blocks]: the CTA that begins the item
  int* status;
};

// One query row: request, token and query head.  Row i of a tile is query head
// kh * group + i % group of token i / group.
struct Row {
  int r, m, h;
  bool live;
};

__device__ __forceinline__ int64_t row_index(const Params& p, const Row& w) {
  return ((int64_t)w.r * p.queries + w.m) * p.heads + w.h;
}
__device__ __forceinline__ int own_length(const Params& p, int r) {
  return p.own_len ? min(max(__ldg(p.own_len + r), 0), p.cache) : p.cache;
}
__device__ __forceinline__ int query_count(const Params& p, int r) {
  return p.q_len ? min(max(__ldg(p.q_len + r), 0), p.queries) : p.queries;
}

// Finite biases count as at most this much, either way.  Both kernels keep it: at
// every scale that tc_kernel takes, the bias over the scale stays inside fp32.
constexpr float kBiasLimit = 1e30f;
constexpr float kLeastScale = 1e-6f, kMostScale = 1e6f;

// What the sum of a row's first partial output holds when its output is written.
constexpr float kWritten = -1.0f;

// Units of time that a step of tc_kernel counts, with rows in two tiles (1.36 us at
// head_dim 64, 2.4 at 128) or in one (1.11, 1.9), and the steps that beginning and
// ending an item are worth.
constexpr int kPair = 5, kSingle = 4, kItemSteps = 2;

// The tensor-core kernel's share of a call: 128-row tiles over the prefix and,
// unless `fold`, each request's own keys.
struct TcPlan {
  int fold;      // rows run through all requests (prefix only), else within one request
  int tokens;    // tokens a tile's rows may come from: requests * queries (fold) or queries
  int per_tile;  // tokens of a 128-row tile
  int tiles;     // of the tokens
  int blocks;    // tiles of all key heads (and requests)
  int halves;    // every item has rows in one tile only
  int ctas;      // each takes a span of the units of work
  int least;     // of at least so many: no item is cut into more than `slots` parts
  int slots;
  int keep;      // chunks of rows_kernel join in: also items that are not cut leave their outputs,
                 // two fp32 rows for each of bf16 (200 x 1,374 tokens over 66,845 + 1,374 keys: 2.4 GB and
                 // 109 ms; the joint form would take 0.1 GB and 118 ms)
};

// Where the output of an item's part lies.  A CTA's span begins inside at most one
// item and ends inside at most one, so that its parts have two places (and two row
// tiles each), whatever the number of rows; `first` parts lie by row tile where
// uncut items leave theirs too.
__host__ __device__ inline int64_t part_tiles(const TcPlan& tc) {
  return (tc.keep ? tc.blocks : tc.ctas * (tc.halves ? 1 : 2)) + (int64_t)tc.ctas * (tc.halves ? 1 : 2);
}
__device__ __forceinline__ int64_t part_tile(const TcPlan& tc, int block, int second, int cta, bool first) {
  if (tc.keep && first) return block;
  const int per = tc.halves ? 1 : 2;
  return (tc.keep ? tc.blocks : first ? tc.ctas * per : 0) + (int64_t)cta * per + second;
}

// Row i of row tile `block` of tc_kernel.
__device__ __forceinline__ Row tile_row(const Params& p, const TcPlan& tc, int kh, int req, int tile, int i) {
  Row w;
  const int tl = i / p.group, tok = tile * tc.per_tile + tl;
  w.h = kh * p.group + (i - tl * p.group);
  w.live = tl < tc.per_tile && tok < tc.tokens;
  w.r = req;
  w.m = tok;
  if (tc.fold) {
    w.r = tok / p.queries;
    w.m = tok - w.r * p.queries;
  }
  if (w.live && p.q_len) w.live = w.m < __ldg(p.q_len + w.r);
  return w;
}

// Whether the kernel can take the call's strides and scale.
bool tc_takes(const Params& p, int head_dim, bool fold);
int launch_tc(const Params& p, int head_dim, const TcPlan& t, cudaStream_t st);

}  // namespace prefix
}  // namespace gpa
