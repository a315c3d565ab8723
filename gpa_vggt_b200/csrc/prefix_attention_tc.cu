// Attention over a shared prefix and own keys for many query rows, on the
// 5th-generation tensor cores (see prefix_attention.cu for the call).
//
// An item is a pair of 128-row tiles of one key/value head and all of its key
// tiles: the prefix's, then the request's own ones, in one online softmax.  One
// CTA per SM; the items' key tiles, laid end to end, are dealt out in equal spans,
// so that a CTA may begin and end inside an item (its part is joined later) and
// no wave is left half empty: the lengths on the device set the spans.  Calls of
// which every item has rows in one tile only (HALVES) run it over the even and the
// odd key tiles at once instead; elsewhere the softmax of the tile that an item may
// lack at its end is left out.  384 threads:
//   warp 0     TMA producer: Q, then K and V tiles of 128 keys through a ring
//              each, on into the next item; writes a tile's bias / scale as three
//              bf16 terms (24 bits) that one more K=16 step adds to the scores,
//              -inf for keys that are out.
//   warps 1-2  MMA issuers, one per stream (row tile, or half of the key tiles):
//              S = Q K^T (+ bias), O += P V with P from TMEM.  Before a tile's
//              first product they zero the K and V rows of keys that are out (past
//              a request's length, or -inf in the bias), whose memory may hold
//              anything.
//   warp 3     works out the CTA's pieces ahead of the others and hands them on in
//              a small ring.
//   warps 4-11 two softmax warpgroups, one per stream, a thread per row: S from
//              TMEM, running maximum that moves only by more than 2^8, P back as
//              bf16.
// At head_dim 64 S, P and O of both streams fit TMEM side by side and S(j+1) runs
// during the softmax of S(j).  At 128 P(j) takes the columns of S(j), and S(j+1)
// waits for O += P(j) V; the other stream's softmax runs meanwhile.
//
// Bound by the softmax at head_dim 64 (issue slots and MUFU: 50% and 55% busy, the
// tensor pipe 40%) and by the issuers' round trip at 128.  Whole tiles (9,472 rows
// x 16,384 keys, replayed from a graph, by card and power): 840-865 TFLOP/s for 16
// heads of 64 (780-834 with a bias), 930-1,095 for 8 of 128.  Four requests of 1,374
// tokens over 16,711 + 1,374 keys: 540-550 us (one CTA per item 685: 384 items end in
// a third of a wave).  In halves 64 rows over 66,845 keys take 76-79 us with the join,
// 128 rows 77-80: 7 us until the first scores, then 1.95 a key tile and stream (77%
// of the measured copy rate).
#include "prefix_attention.cuh"

namespace gpa {
namespace prefix {

constexpr int TC_THREADS = 384;
constexpr int TM = 128;   // rows and keys per tile
constexpr int XTILE = TM * 16 * 2;
// c*x - c*m is off by the rounding of c*m, the same for all of a row's keys.  Up to
// this maximum (log2 units) that is at most 64 and stays inside the exponent's range.
// Beyond it (large biases, or nothing but the type's lowest value) scores that differ
// at all differ by 64 or more, so that only keys at the maximum count, and any factor
// near c gives the same weights: such a row takes c's power of two, whose products are
// exact.  (Taking m off x first costs every row: 612 us for 549 at 4 x 1,374 tokens.)
constexpr float kFar = 1073741824.f;
constexpr int TC_REGS = 168, TC_LOW = 80, TC_HIGH = 208;
static_assert(TC_LOW * 128 + TC_HIGH * 256 <= TC_REGS * TC_THREADS, "register split");

constexpr int RING = 4;   // pieces handed on ahead

template <int D, bool HALVES>
struct TcSmem {
  static constexpr int ATOMS = D / 64;           // a row is ATOMS swizzled rows of 128 bytes
  static constexpr int ATOM = TM * 128;          // 16 KB
  static constexpr int TILE = ATOMS * ATOM;
  // In halves each stage belongs to one stream (an even number of them): an issuer
  // sees every phase of the barriers that it waits on.
  static constexpr int STAGES = D == 64 ? (HALVES ? 4 : 3) : 2;
  static_assert(!HALVES || STAGES % 2 == 0, "stages of the two streams");
  static constexpr int Q = 0;                    // 1 or 2 tiles
  static constexpr int K = Q + (HALVES ? 1 : 2) * TILE;
  static constexpr int V = K + STAGES * TILE;
  static constexpr int ONES = V + STAGES * TILE;
  static constexpr int BETA = ONES + XTILE;
  static constexpr int MASK = BETA + STAGES * XTILE;   // 4 words per key tile, twice as many as stages: V is used
  static constexpr int ML = MASK + 2 * STAGES * 16;    // after its K's stage has gone on; the second stream's maxima and sums
  static constexpr int BARS = ML + TM * 8;
  static constexpr int TOTAL = BARS + 384;
  static constexpr int ALLOC = TOTAL + 1024;
  static_assert((4 + 4 * STAGES + 8 + 2 * RING) * 8 + 8 <= 384, "barrier area");
  static_assert(ALLOC <= 232448, "shared memory per CTA");
};

__host__ __device__ constexpr int xtile_off(int row, int k) {
  return (row >> 3) * 256 + (k >> 3) * 128 + (row & 7) * 16 + (k & 7) * 2;
}

// no-swizzle K-major descriptor of a bias tile: 8x8 core matrices, K halves 128 B
// apart, row groups 256 B apart
__device__ __forceinline__ uint64_t sdesc_plain(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | static_cast<uint64_t>(128 >> 4) << 16 |
         static_cast<uint64_t>(256 >> 4) << 32 | static_cast<uint64_t>(1) << 46;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2 of 8 exponentials on the FMA pipe, the rest on MUFU.  The cubic is off by up to
// 7.7e-5: fifty times less than P's rounding to bf16, but the row sum carries it, so
// lse is off by up to 1.1e-4 where such a key dominates.  Weights below 2^-126 count
// as that in these two.
__device__ __forceinline__ void exp8(const float* x, float* e) {
#pragma unroll
  for (int i = 0; i < 6; ++i) e[i] = fast_exp2(x[i]);
  exp2_poly2<3>(x[6], x[7], e[6], e[7]);
}

// The order of work: requests, their key heads, the head's row-tile pairs, a
// pair's steps (a key tile; two of them in halves) and kItemSteps more for its
// ends.  A step of a pair with two row tiles counts kPair units, of one kSingle.
struct Load {
  int pairs2;      // pairs with two row tiles
  bool single;     // and one with one
  int steps;       // of a pair (no keys at all count as one, to write the empty rows)
  int head;        // units of one key head
};
template <bool HALVES>
__device__ __forceinline__ Load load_of(const Params& p, const TcPlan& tc, int r) {
  Load w;
  const int tokens = tc.fold ? tc.tokens : query_count(p, r);
  const int tiles = (tokens + tc.per_tile - 1) / tc.per_tile;
  w.pairs2 = tiles >> 1;
  w.single = tiles & 1;
  const int keys = max(1, (p.prefix + TM - 1) / TM + (tc.fold ? 0 : (own_length(p, r) + TM - 1) / TM));
  w.steps = HALVES ? (keys + 1) >> 1 : keys;
  w.head = (w.steps + kItemSteps) * (kPair * w.pairs2 + (w.single ? kSingle : 0));
  return w;
}

// A CTA's share of one item.
struct Piece {
  int req, kh, tile;   // the first of its two row tiles
  int len, qlen;
  int j0, nk;        // key tiles (nk may be 0: nothing to see here)
  int slot;          // which partial output
  bool first, last;  // holds the item's first, last step
  bool single;       // the second row tile has no rows
};
// A piece from shared memory, read anew at each call: what the softmax needs after
// its key tiles does not stay in registers meanwhile (a few more of them made its
// loop 15% slower).
__device__ __forceinline__ Piece read_piece(const Piece* at) {
  const volatile Piece* v = at;
  Piece c;
  c.req = v->req; c.kh = v->kh; c.tile = v->tile;
  c.len = v->len; c.qlen = v->qlen;
  c.j0 = v->j0; c.nk = v->nk;
  c.slot = v->slot;
  c.first = v->first; c.last = v->last;
  c.single = v->single;
  return c;
}
struct Walk {
  int pos, end, span;   // this CTA's units (all of a call's fit 31 bits)
  int req;
  int req0;             // first unit of the request
};
template <bool HALVES>
__device__ __forceinline__ bool next_piece(const Params& p, const TcPlan& tc, Walk& w, Piece& c) {
  int a, b, steps;
  do {
    if (w.pos >= w.end) return false;
    Load ld = load_of<HALVES>(p, tc, w.req);
    while (w.pos - w.req0 >= ld.head * p.kv_heads) {
      w.req0 += ld.head * p.kv_heads;
      ld = load_of<HALVES>(p, tc, ++w.req);
    }
    const int x = w.pos - w.req0;
    c.kh = x / ld.head;
    const int y = x - c.kh * ld.head;
    steps = ld.steps;
    const int whole = kPair * (steps + kItemSteps), pair = min(y / whole, ld.pairs2);
    const int at = y - pair * whole;   // units of the pair that others have
    const int each = pair < ld.pairs2 ? kPair : kSingle;
    const int units = min((steps + kItemSteps) * each - at, w.end - w.pos);
    // a step goes to the CTA that has its first unit
    a = min(steps, (at + each - 1) / each);
    b = min(steps, (at + units + each - 1) / each);
    c.slot = blockIdx.x - (w.pos - at) / w.span;
    c.tile = pair * 2;
    c.single = each == kSingle;
    w.pos += units;
  } while (a == b);   // the rest of a step, or of an item, that the CTA before has done
  c.req = w.req;
  c.qlen = tc.fold ? p.queries : query_count(p, c.req);
  c.len = tc.fold ? 0 : own_length(p, c.req);
  // with an order, no row of this pair sees an own key from here on
  const int own_end =
      p.causal ? min(c.len, max(0, c.len - c.qlen + min((c.tile + 2) * tc.per_tile, c.qlen))) : c.len;
  const int tiles = (p.prefix + TM - 1) / TM + (own_end + TM - 1) / TM, each = HALVES ? 2 : 1;
  c.j0 = a * each;
  c.nk = max(0, min(tiles, b * each) - c.j0);
  c.first = a == 0;
  c.last = b == steps;
  return true;
}

// CAUSAL: own keys in order (a kernel of its own: the mask costs the others registers).
template <int D, bool CAUSAL, bool HALVES>
__global__ void __launch_bounds__(TC_THREADS, 1)
    tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kp,
              const __grid_constant__ CUtensorMap map_vp, const __grid_constant__ CUtensorMap map_ko,
              const __grid_constant__ CUtensorMap map_vo, const Params p, const TcPlan tc) {
  using SM = TcSmem<D, HALVES>;
  constexpr int ST = SM::STAGES;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ int warp_units[TC_THREADS / 32];
  __shared__ int start_req0, start_req;
  __shared__ Piece ring[RING];
  asm volatile("griddepcontrol.launch_dependents;");   // the join may be launched, and waits for this grid's end
  const int warp = warp_id(), lane = lane_id();

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + SM::BARS);
  uint64_t* q_empty = q_full + 1;      // both streams' score products of the item are done
  uint64_t* k_full = q_empty + 1;
  uint64_t* v_full = k_full + ST;
  uint64_t* k_empty = v_full + ST;
  uint64_t* v_empty = k_empty + ST;
  uint64_t* s_full = v_empty + ST;     // 2
  uint64_t* s_empty = s_full + 2;      // 2
  uint64_t* p_full = s_empty + 2;      // 2
  uint64_t* o_done = p_full + 2;       // 2
  uint64_t* half_there = o_done + 2;   // the second stream's half is complete
  uint64_t* half_read = half_there + 1;
  uint64_t* piece_full = half_read + 1;      // RING
  uint64_t* piece_empty = piece_full + RING;   // RING
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(piece_empty + RING);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  // All units, this CTA's span of them, and the request that it starts in: each
  // thread adds up a run of requests.
  Walk walk;
  const int nreq = tc.fold ? 1 : p.requests;
  const int run = (nreq + TC_THREADS - 1) / TC_THREADS;
  const int r0 = threadIdx.x * run, r1 = min(nreq, r0 + run);
  int mine = 0;
  for (int r = r0; r < r1; ++r) mine += load_of<HALVES>(p, tc, r).head * p.kv_heads;
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) warp_units[warp] = upto;

  // Every barrier's phases run on through the CTA's pieces: per role, `g` counts
  // the key tiles of all pieces so far, `c` those of one stream, `i` the pieces
  // that have key tiles.
  if (threadIdx.x == 0) {
    bar_init(q_full, 1);
    bar_init(q_empty, 2);
    for (int s = 0; s < ST; ++s) {
      bar_init(&k_full[s], 1);
      bar_init(&v_full[s], 1);
      bar_init(&k_empty[s], HALVES ? 1 : 2);   // one arrival per row tile
      bar_init(&v_empty[s], HALVES ? 1 : 2);
    }
    for (int t = 0; t < 2; ++t) {
      bar_init(&s_full[t], 1);
      bar_init(&s_empty[t], 4);
      bar_init(&p_full[t], 4);
      bar_init(&o_done[t], 1);
    }
    for (int s = 0; s < RING; ++s) {
      bar_init(&piece_full[s], 1);
      bar_init(&piece_empty[s], 11);   // producer, issuers, softmax warps
    }
    bar_init(half_there, 4);
    bar_init(half_read, 4);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_kp);
    tma_prefetch_desc(&map_vp);
    tma_prefetch_desc(&map_ko);
    tma_prefetch_desc(&map_vo);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tmem_slot;
  {
    int before = 0, total = 0;
#pragma unroll
    for (int i = 0; i < TC_THREADS / 32; ++i) {
      if (i < warp) before += warp_units[i];
      total += warp_units[i];
    }
    walk.span = max((int)((total + gridDim.x - 1) / gridDim.x), tc.least);
    walk.pos = min((int64_t)blockIdx.x * walk.span, (int64_t)total);
    walk.end = min((int64_t)walk.pos + walk.span, (int64_t)total);
    int at = before + upto - mine;
    if (walk.pos >= at && walk.pos < at + mine) {
      int r = r0;
      for (;; ++r) {
        const int n = load_of<HALVES>(p, tc, r).head * p.kv_heads;
        if (walk.pos < at + n) break;
        at += n;
      }
      start_req = r;
      start_req0 = at;
    }
    __syncthreads();
  }
  const int tp = (p.prefix + TM - 1) / TM;
  auto wait = [&](uint64_t* bar, uint32_t phase) {   // the whole warp, bounded
    return __all_sync(0xffffffffu, wait_bar(bar, phase & 1, abort_flag, p.status, kDevTimeout)) != 0;
  };
  // The next piece of the ring (`turn` counts them) into c, or false at the end;
  // done() gives its place back.
  auto next = [&](Piece& c, uint32_t turn, bool& okw) {
    okw = wait(&piece_full[turn % RING], turn / RING);
    if (!okw) return false;
    c = read_piece(&ring[turn % RING]);
    return c.req >= 0;
  };
  auto done = [&](uint32_t turn) {
    __syncwarp();
    if (lane == 0) bar_arrive(&piece_empty[turn % RING]);
  };
  // key tile j of a piece: the prefix's or an own one
  struct Tile {
    bool own;
    int key0, valid;   // keys of the tile that exist
  };
  auto tile_of = [&](const Piece& c, int j) {
    Tile t;
    t.own = c.j0 + j >= tp;
    t.key0 = (t.own ? c.j0 + j - tp : c.j0 + j) * TM;
    t.valid = min(TM, (t.own ? c.len : p.prefix) - t.key0);
    return t;
  };
  auto has_beta = [&](const Tile& t) { return t.valid < TM || (!t.own && p.bias != nullptr); };
  // key tiles of stream t, and which they are (g: all earlier pieces' key tiles)
  auto tiles_of = [](const Piece& c, int t, int g) { return HALVES ? (c.nk - ((t - g) & 1) + 1) >> 1 : c.nk; };
  auto key_tile = [](int t, int j, int g) { return HALVES ? 2 * j + ((t - g) & 1) : j; };
  // TMEM columns of a stream
  auto col_s = [](int t) { return (uint32_t)(t * TM); };
  auto col_o = [](int t) { return (uint32_t)(256 + t * D); };
  auto col_p = [](int t) { return (uint32_t)(D == 64 ? 384 + t * 64 : t * TM); };

  if (warp < 4) {
    regs_dec<TC_LOW>();
    if (warp == 0) {
      // ------------------------------ producer ------------------------------
      uint32_t* w = reinterpret_cast<uint32_t*>(smem + SM::ONES);
      for (int i = lane; i < XTILE * (1 + ST) / 4; i += 32) w[i] = 0u;
      __syncwarp();
      for (int row = lane; row < TM; row += 32)   // 1, 1, 1, 0, ...
        *reinterpret_cast<uint2*>(smem + SM::ONES + xtile_off(row, 0)) = make_uint2(0x3F803F80u, 0x3F80u);
      fence_async_smem();
      const float inv_scale = 1.0f / p.scale, most = kBiasLimit * inv_scale;
      int i = 0, gk = 0, gv = 0;
      bool okw = true;
      Piece c;
      for (uint32_t turn = 0; okw && next(c, turn, okw); ++turn) {
        done(turn);
        if (c.nk == 0) continue;
        if (i > 0 && !(okw = wait(q_empty, i - 1))) break;
        if (lane == 0) {
          constexpr int TILES = HALVES ? 1 : 2;   // past the last token the copy fills with zeros
          bar_expect_tx(q_full, TILES * SM::ATOMS * p.group * tc.per_tile * 128);
          for (int t = 0; t < TILES; ++t)
            for (int h = 0; h < SM::ATOMS; ++h)
              tma_load_4d(&map_q, q_full, smem + SM::Q + t * SM::TILE + h * SM::ATOM, h * 64, c.kh * p.group,
                          (c.tile + t) * tc.per_tile, c.req);
        }
        ++i;
        const float* brow = p.bias ? p.bias + c.kh * p.bias_sh : nullptr;
        float braw[4];
        auto load_bias = [&](int j) {   // raw bias of a tile, one tile ahead of its use
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int key = (c.j0 + j) * TM + u * 32 + lane;
            braw[u] = (brow && c.j0 + j < tp && key < p.prefix) ? __ldg(brow + key) : 0.f;
          }
        };
        load_bias(0);
        for (int j = 0; j < c.nk; ++j) {
          const int s = gk % ST;
          const uint32_t ph = gk / ST;
          const Tile t = tile_of(c, j);
          if (!(okw = wait(&k_empty[s], ph + 1))) break;
          if (has_beta(t)) {
            uint32_t* mask = reinterpret_cast<uint32_t*>(smem + SM::MASK + gk % (2 * ST) * 16);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int row = u * 32 + lane;
              const bool in = row < t.valid && braw[u] > -INFINITY;   // NaN takes a key out too
              const float beta = in ? fminf(fmaxf(braw[u] * inv_scale, -most), most) : -INFINITY;
              const __nv_bfloat16 hi = __float2bfloat16_rn(beta);
              float rest = in ? beta - __bfloat162float(hi) : 0.f;
              const __nv_bfloat16 mid = __float2bfloat16_rn(rest);
              rest -= __bfloat162float(mid);
              *reinterpret_cast<uint2*>(smem + SM::BETA + s * XTILE + xtile_off(row, 0)) = make_uint2(
                  (uint32_t)__bfloat16_as_ushort(hi) | (uint32_t)__bfloat16_as_ushort(mid) << 16,
                  (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(rest)));
              // rows to zero: own ones past the length, prefix ones by their bias
              // (past the prefix's end the copy fills with zeros)
              const unsigned out = __ballot_sync(0xffffffffu, !in && (t.own || row < t.valid));
              if (lane == 0) mask[u] = out;
            }
            fence_async_smem();
            __syncwarp();
          }
          load_bias(j + 1);
          if (lane == 0) {
            bar_expect_tx(&k_full[s], SM::TILE);
            for (int h = 0; h < SM::ATOMS; ++h)
              tma_load_4d(t.own ? &map_ko : &map_kp, &k_full[s], smem + SM::K + s * SM::TILE + h * SM::ATOM, h * 64,
                          t.key0, c.kh, t.own ? c.req : 0);
          }
          ++gk;
          if (!(okw = wait(&v_empty[s], ph + 1))) break;
          if (lane == 0) {
            bar_expect_tx(&v_full[s], SM::TILE);
            for (int h = 0; h < SM::ATOMS; ++h)
              tma_load_4d(t.own ? &map_vo : &map_vp, &v_full[s], smem + SM::V + s * SM::TILE + h * SM::ATOM, h * 64,
                          t.key0, c.kh, t.own ? c.req : 0);
          }
          ++gv;
        }
      }
      if (lane == 0) {   // copies in flight land before the CTA exits
        const unsigned long long t0 = global_ns();
        if (i > 0) drain_bar(q_full, (i - 1) & 1, t0);
        for (int j = max(0, gk - ST); j < gk; ++j) drain_bar(&k_full[j % ST], (j / ST) & 1, t0);
        for (int j = max(0, gv - ST); j < gv; ++j) drain_bar(&v_full[j % ST], (j / ST) & 1, t0);
      }
    } else if (warp < 3) {
      // ------------------------------ MMA issuers ------------------------------
      const int t = warp - 1;
      const bool leader = elect_one();
      constexpr uint32_t idesc_s = idesc_bf16(TM, TM, false, false);
      constexpr uint32_t idesc_o = idesc_bf16(TM, D, false, true);
      const uint64_t dQ0 = sdesc_sw128(smem_u32(smem + SM::Q), 16, 1024);
      const uint64_t dK = sdesc_sw128(smem_u32(smem + SM::K), 16, 1024);
      const uint64_t dV = sdesc_sw128(smem_u32(smem + SM::V), SM::ATOM, 1024);
      const uint64_t dOnes = sdesc_plain(smem_u32(smem + SM::ONES));
      const uint64_t dBeta = sdesc_plain(smem_u32(smem + SM::BETA));
      const uint32_t dS = tbase + col_s(t), dO = tbase + col_o(t), dP = tbase + col_p(t);
      // What follows a softmax's signal is kept short: the next tile's K, its bias
      // and its rows to zero are seen to before.
      int i = 0, g = 0, cs = 0;   // cs: this stream's key tiles in earlier pieces
      constexpr int STEP = HALVES ? 2 : 1;
      int kst = HALVES ? t : 0, vst = kst;   // this stream's next K and V stage, and their phases
      uint32_t kph = 0, vph = 0;
      bool okw = true;
      // Zeroes the rows of key tile gt (of all pieces) that are out.  Where both
      // issuers read a tile, the second writes the same zeros.
      auto zero_rows = [&](int gt, uint8_t* tile) {
        const uint4 m = *reinterpret_cast<const uint4*>(smem + SM::MASK + gt % (2 * ST) * 16);
        if (!(m.x | m.y | m.z | m.w)) return;
        tile += (lane >> 3) * SM::ATOM + (lane & 7) * 16;
        for (int row = 0; row < TM; ++row) {
          const uint32_t word = row < 64 ? (row < 32 ? m.x : m.y) : (row < 96 ? m.z : m.w);
          if ((word >> (row & 31) & 1) && lane < 8 * SM::ATOMS)
            *reinterpret_cast<uint4*>(tile + row * 128) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_async_smem();
        __syncwarp();
      };
      auto run = [&](const Piece& c) {
        const int n = tiles_of(c, t, g);
        const uint64_t dQ = dQ0 + (uint64_t)((HALVES ? 0 : t) * (SM::TILE >> 4));
        bool beta = false;
        auto k_landed = [&](int j) {
          const int jt = key_tile(t, j, g);
          const Tile kt = tile_of(c, jt);
          beta = has_beta(kt);
          if (!wait(&k_full[kst], kph)) return false;
          if (kt.own ? kt.valid < TM : p.bias != nullptr) zero_rows(g + jt, smem + SM::K + kst * SM::TILE);
          return true;
        };
        auto v_landed = [&](int j) {
          const int jt = key_tile(t, j, g);
          const Tile kt = tile_of(c, jt);
          if (!wait(&v_full[vst], vph)) return false;
          if (kt.own ? kt.valid < TM : p.bias != nullptr) zero_rows(g + jt, smem + SM::V + vst * SM::TILE);
          return true;
        };
        auto issue_s = [&](bool last) {
          tc_fence_after();
          if (leader) {
            const uint64_t bk = dK + (uint64_t)(kst * (SM::TILE >> 4));
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint64_t off = (uint64_t)((k >> 2) * (SM::ATOM >> 4) + (k & 3) * 2);
              umma_bf16(dS, dQ + off, bk + off, idesc_s, k != 0);
            }
            if (beta) umma_bf16(dS, dOnes, dBeta + (uint64_t)(kst * (XTILE >> 4)), idesc_s, 1);
            umma_commit(&s_full[t]);
            umma_commit(&k_empty[kst]);
            if (last) umma_commit(q_empty);
          }
          __syncwarp();
          kst += STEP;
          if (kst >= ST) {
            kst -= ST;
            kph ^= 1;
          }
        };
        auto issue_o = [&](bool first) {
          tc_fence_after();
          if (leader) {
            const uint64_t bv = dV + (uint64_t)(vst * (SM::TILE >> 4));
#pragma unroll
            for (int ks = 0; ks < TM / 16; ++ks)
              umma_bf16_ts(dO, dP + ks * 8, bv + (uint64_t)(ks * (2048 >> 4)), idesc_o, (!first || ks > 0));
            umma_commit(&o_done[t]);
            umma_commit(&v_empty[vst]);
          }
          __syncwarp();
          vst += STEP;
          if (vst >= ST) {
            vst -= ST;
            vph ^= 1;
          }
        };
        okw = wait(q_full, i);
        if (okw && n == 0 && leader) bar_arrive(q_empty);   // nothing to read for this stream
        if (!HALVES && t == 1 && c.single) {   // no rows: only the barriers go on
          for (int j = 0; okw && j < n; ++j) {
            okw = wait(&k_full[kst], kph);
            if (!okw) break;
            if (leader) {
              bar_arrive(&s_full[t]);
              bar_arrive(&k_empty[kst]);
              if (j == n - 1) bar_arrive(q_empty);
            }
            kst = kst + 1 == ST ? 0 : kst + 1;
            kph ^= kst == 0;
            okw = wait(&p_full[t], cs + j) && wait(&v_full[vst], vph);
            if (!okw) break;
            if (leader) {
              bar_arrive(&o_done[t]);
              bar_arrive(&v_empty[vst]);
            }
            vst = vst + 1 == ST ? 0 : vst + 1;
            vph ^= vst == 0;
          }
          cs += n;
          return;
        }
        if (okw && n > 0) {
          // S is free once the last softmax has read it, or (P in its place) the last product with V is done
          okw = k_landed(0) && (cs == 0 || wait(D == 64 ? &s_empty[t] : &o_done[t], cs - 1));
          if (okw) issue_s(n == 1);
        }
        for (int j = 0; okw && j < n; ++j) {
          const bool more = j + 1 < n;
          okw = v_landed(j) && (!more || k_landed(j + 1));
          if (!okw) break;
          if (D == 64) {
            if (more) {
              if (!(okw = wait(&s_empty[t], cs + j))) break;
              issue_s(j + 2 == n);
            }
            if (!(okw = wait(&p_full[t], cs + j))) break;
            issue_o(j == 0);
          } else {
            if (!(okw = wait(&p_full[t], cs + j))) break;
            issue_o(j == 0);
            if (more) {   // S(j+1) overwrites P(j), which O += P(j) V still reads until it is done
              if (!(okw = wait(&o_done[t], cs + j))) break;
              issue_s(j + 2 == n);
            }
          }
        }
        cs += n;
      };
      Piece c;
      for (uint32_t turn = 0; okw && next(c, turn, okw); ++turn) {
        done(turn);
        if (c.nk == 0) continue;
        run(c);
        ++i;
        g += c.nk;
      }
    } else {
      // ------------------------------ planner ------------------------------
      walk.req = start_req;
      walk.req0 = start_req0;
      Piece c;
      for (uint32_t turn = 0;; ++turn) {
        const bool more = next_piece<HALVES>(p, tc, walk, c);
        if (!wait(&piece_empty[turn % RING], turn / RING + 1)) break;
        if (lane == 0) {
          if (!more) c.req = -1;
          ring[turn % RING] = c;
          bar_arrive(&piece_full[turn % RING]);
        }
        if (!more) break;
      }
    }
  } else {
    regs_inc<TC_HIGH>();
    // ------------------------------ softmax ------------------------------
    const int t = (warp - 4) >> 2;
    const int quad = warp & 3;
    const int row_i = quad * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const uint32_t tS = tbase + lane_off + col_s(t), tO = tbase + lane_off + col_o(t), tP = tbase + lane_off + col_p(t);
    float2* half_ml = reinterpret_cast<float2*>(smem + SM::ML) + row_i;
    const float c2 = p.scale_log2, c2_pow2 = __uint_as_float(__float_as_uint(c2) & 0x7f800000u);
    constexpr float kNoMax = -3.0e38f;   // no key yet
    int cs = 0, g = 0, ih = 0;   // ih: pieces in halves so far
    bool okw = true;
    auto run = [&](const Piece& c0, const Piece* at) {
      const int n = tiles_of(c0, t, g);
      bool live;
      int limit;   // own keys that this row sees end here
      {
        const Row row = tile_row(p, tc, c0.kh, c0.req, c0.tile + (HALVES ? 0 : t), row_i);
        live = row.live;
        limit = CAUSAL ? c0.len - c0.qlen + row.m + 1 : 0;
      }
      const bool idle = !__any_sync(0xffffffffu, live);   // a warp without rows only keeps the barriers going
      float m_raw = kNoMax, l = 0.f;       // running maximum (score units), row sum
      float cr = c2, neg_mc = 0.f;         // the row's factor, and -cr * m_raw
      // For each tile at head_dim 64, where the maximum moves at 128: the other way round
      // four frames take 577 us for 549, 9,472 rows x 16,384 keys 740 for 693 at 128.
      auto set_factor = [&] {
        cr = fabsf(m_raw * c2) > kFar ? c2_pow2 : c2;
        neg_mc = -m_raw * cr;
        if (D == 64) neg_mc = fminf(neg_mc, -kNoMax);   // of a row without a key yet: finite
      };
      auto quarter = [&](float* xq, float* acc, uint32_t* pk) {
#pragma unroll
        for (int e8 = 0; e8 < 4; ++e8) {
          float* xg = xq + e8 * 8;
#pragma unroll
          for (int i = 0; i < 8; i += 2) ffma2(xg[i], xg[i + 1], xg[i], xg[i + 1], cr, cr, neg_mc, neg_mc);
          float e[8];
          exp8(xg, e);
#pragma unroll
          for (int i = 0; i < 8; i += 2) fadd2(acc[i], acc[i + 1], acc[i], acc[i + 1], e[i], e[i + 1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) pk[e8 * 4 + i] = pack_bf16x2(e[2 * i], e[2 * i + 1]);
        }
      };
      if (idle) {
        for (int j = 0; j < n; ++j) {
          // The next S may be there before the issuer has taken this P: its product
          // must be done, or the issuer could miss a phase of p_full.
          okw = wait(&s_full[t], cs + j) && (cs + j == 0 || wait(&o_done[t], cs + j - 1));
          if (!okw) break;
          if (lane == 0) {
            if (D == 64) bar_arrive(&s_empty[t]);
            bar_arrive(&p_full[t]);
          }
        }
      }
      for (int j = idle ? n : 0; j < n; ++j) {
        if (!wait(&s_full[t], cs + j)) { okw = false; break; }
        tc_fence_after();
        float x[TM];
#pragma unroll
        for (int u = 0; u < TM / 32; ++u) tmem_ld32f(tS + u * 32, x + u * 32);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (D == 64 && lane == 0) bar_arrive(&s_empty[t]);
        if (CAUSAL) {   // keys ahead of this row
          const Tile kt = tile_of(read_piece(at), key_tile(t, j, g));
          if (kt.own && __any_sync(0xffffffffu, limit < kt.key0 + TM)) {
            const int end = limit - kt.key0;
#pragma unroll
            for (int u = 0; u < TM; ++u)
              if (u >= end) x[u] = -INFINITY;
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int u = 0; u < TM / 4; ++u) {
          mx[u & 3] = max3_nan(mx[u & 3], x[4 * u + 0], x[4 * u + 1]);
          mx[u & 3] = max3_nan(mx[u & 3], x[4 * u + 2], x[4 * u + 3]);
        }
        const float mt = max3_nan(max3_nan(mx[0], mx[0], mx[1]), mx[2], mx[3]);
        float alpha = 1.f;
        // the maximum moves: also the first time, and for a NaN (never for a row without keys)
        const bool moved = live && !((mt - m_raw) * c2 <= 8.0f);
        const bool any_moved = __any_sync(0xffffffffu, moved);
        if (any_moved) {
          if (moved) {
            alpha = fast_exp2((m_raw - mt) * c2);
            l = mt < INFINITY ? l * alpha : NAN;   // a NaN or infinite score: the row is NaN (the polynomial would lose it)
            m_raw = mt < INFINITY ? mt : 0.f;
            if (D == 128) set_factor();
          }
        }
        if (D == 64) set_factor();
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        uint32_t pk[4][16];
#pragma unroll
        for (int qt = 0; qt < 4; ++qt) {
          quarter(x + qt * 32, acc, pk[qt]);
          if (D == 128) {   // S(j) came after O += P(j-1) V
            tmem_st16(tP + qt * 16, pk[qt]);
          } else if (qt == 1) {
            if (j > 0) {    // P and O are busy until O += P(j-1) V is done
              if (!wait(&o_done[t], cs + j - 1)) { okw = false; break; }
              tc_fence_after();
            }
            tmem_st16(tP, pk[0]);
            tmem_st16(tP + 16, pk[1]);
          } else if (qt > 1) {
            tmem_st16(tP + qt * 16, pk[qt]);
          }
        }
        if (!okw) break;
        l += ((acc[0] + acc[1]) + (acc[2] + acc[3])) + ((acc[4] + acc[5]) + (acc[6] + acc[7]));
        if (j > 0 && any_moved) {
          uint32_t ov[32];
#pragma unroll
          for (int u = 0; u < D / 32; ++u) {
            tmem_ld32(tO + u * 32, ov);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
            tmem_st32(tO + u * 32, ov);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&p_full[t]);
      }
      const Piece c = read_piece(at);
      const bool halves = HALVES && c.nk > 0, other = halves && tiles_of(c, 1, g) > 0;
      cs += n;
      g += c.nk;
      if (okw && n > 0) okw = wait(&o_done[t], cs - 1);
      tc_fence_after();
      if (halves && t == 1) {   // hand over this half: O stays in TMEM until it is read
        if (okw) {
          *half_ml = make_float2(m_raw, l);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(half_there);
          okw = wait(half_read, ih);
        }
        ++ih;
        return;
      }
      if (HALVES && t == 1) return;
      float f0 = 1.f, f1 = 0.f;
      if (halves) {
        okw = okw && wait(half_there, ih);
        ++ih;
        if (okw) {
          tc_fence_after();
          const float2 ml = *half_ml;
          const float m = fmaxf(m_raw, ml.x);
          f0 = fast_exp2((m_raw - m) * c2);
          f1 = fast_exp2((ml.x - m) * c2);
          l = l * f0 + ml.y * f1;
          m_raw = m;
        }
      }
      if (!okw || *abort_flag) return;
      const bool some = m_raw > kNoMax;   // else the sum holds the polynomial's 2^-126
      const float inv = some ? 1.0f / l : 0.f;
      const bool direct = c.first && c.last && p.s2 == 0;
      const Row row = tile_row(p, tc, c.kh, c.req, c.tile + (HALVES ? 0 : t), row_i);
      // the row tile among the partial outputs, and in this piece's slot
      const int block = (c.req * p.kv_heads + c.kh) * tc.tiles + c.tile + (HALVES ? 0 : t);
      const int64_t to = (int64_t)c.slot * tc.blocks + block;
      const int64_t part = part_tile(tc, block, HALVES ? 0 : t, blockIdx.x, c.first);
      __nv_bfloat16* orow = p.o + row.r * p.o_sr + row.h * p.o_sh + row.m * p.o_sm;
      if (!idle) {
#pragma unroll
        for (int u = 0; u < D / 32; ++u) {
          float v[32];
          {
            uint32_t ov[32];
            if (n > 0) {
              tmem_ld32(tO + u * 32, ov);
              tmem_wait_ld();
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = n > 0 ? __uint_as_float(ov[i]) : 0.f;
            if (other) {
              tmem_ld32(tbase + lane_off + col_o(1) + u * 32, ov);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = fmaf(v[i], f0, __uint_as_float(ov[i]) * f1);
            }
          }
          if (!row.live) continue;
          if (direct) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = some ? pack_bf16x2(v[2 * i] * inv, v[2 * i + 1] * inv) : 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              reinterpret_cast<uint4*>(orow + u * 32)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
          } else if (some) {
            float4* w = p.tc_o + (part * (D / 4) + u * 8) * TM + row_i;
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i * TM] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          }
        }
      }
      if (halves) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(half_read);
      }
      // (a second tile without rows is another item's, or none)
      if (c.first && !direct && row_i == 0 && (HALVES || t == 0 || !c.single)) p.tc_first[block] = blockIdx.x;
      if (row.live) {
        if (direct) {
          if (p.lse) p.lse[row.r * p.lse_sr + row.h * p.lse_sh + row.m] = some ? m_raw * c2 + log2f(l) : -INFINITY;
          p.tc_ml[(int64_t)block * TM + row_i] = make_float2(0.f, kWritten);
        } else {
          p.tc_ml[to * TM + row_i] = some ? make_float2(m_raw * c2, l) : make_float2(-INFINITY, 0.f);
          if (c.last)   // slots that no piece of this item takes
            for (int s = c.slot + 1; s < tc.slots; ++s)
              p.tc_ml[((int64_t)s * tc.blocks + block) * TM + row_i] = make_float2(-INFINITY, 0.f);
        }
      }
    };
    Piece c;
    for (uint32_t turn = 0; okw && next(c, turn, okw); ++turn) {
      run(c, &ring[turn % RING]);
      done(turn);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

// [batch][mid][rows][head_dim] (strides in elements; a dim of one gets a harmless
// stride), boxes of 64 features x b1 x b2.
static int make_map(CUtensorMap* map, const void* base, int d, int64_t n1, int64_t n2, int64_t n3, int64_t s1,
                    int64_t s2, int64_t s3, int b1, int b2) {
  uint64_t dims[4] = {(uint64_t)d, (uint64_t)n1, (uint64_t)n2, (uint64_t)n3};
  uint64_t st[4] = {2, (uint64_t)s1 * 2, (uint64_t)s2 * 2, (uint64_t)s3 * 2};
  if (n1 == 1) st[1] = (uint64_t)d * 2;
  if (n2 == 1) st[2] = st[1] * (uint64_t)n1;
  if (n3 == 1) st[3] = st[2] * (uint64_t)n2;
  uint32_t box[4] = {64, (uint32_t)b1, (uint32_t)b2, 1};
  return make_map_bf16(map, base, 4, dims, st, box, CU_TENSOR_MAP_SWIZZLE_128B, "gpa_attention_shared_prefix");
}

static bool stride_ok(int64_t n, int64_t s) { return n <= 1 || (s > 0 && s < (1ll << 38)); }

bool tc_takes(const Params& p, int head_dim, bool fold) {
  // the maximum is taken on unscaled scores, and the bias divided by the scale
  if (!(p.scale > kLeastScale && p.scale < kMostScale) || p.group > TM) return false;
  if (!stride_ok(p.heads, p.q_sh) || !stride_ok(p.queries, p.q_sm) || !stride_ok(p.requests, p.q_sr)) return false;
  if (fold && p.requests > 1 && p.queries > 1 && p.q_sr != p.queries * p.q_sm) return false;
  if (p.prefix && (!stride_ok(p.kv_heads, p.kp_sh) || !stride_ok(p.prefix, p.kp_sn) || !stride_ok(p.kv_heads, p.vp_sh) ||
                   !stride_ok(p.prefix, p.vp_sn)))
    return false;
  if (fold || !p.cache) return true;
  return stride_ok(p.requests, p.ko_sr) && stride_ok(p.kv_heads, p.ko_sh) && stride_ok(p.cache, p.ko_sn) &&
         stride_ok(p.requests, p.vo_sr) && stride_ok(p.kv_heads, p.vo_sh) && stride_ok(p.cache, p.vo_sn);
}

// The register split needs a launch with TC_REGS registers per thread; refuse
// to launch otherwise (it would never start).
template <int D, bool CAUSAL, bool HALVES>
static int check_regs() {
  cudaFuncAttributes fa;
  if (cudaFuncGetAttributes(&fa, tc_kernel<D, CAUSAL, HALVES>) != cudaSuccess)
    return fail(GPA_ERR_CUDA, "gpa_attention_shared_prefix: cudaFuncGetAttributes failed");
  if (fa.numRegs * TC_THREADS < TC_LOW * 128 + TC_HIGH * 256)
    return fail(GPA_ERR_CUDA, "gpa_attention_shared_prefix: kernel built with %d registers/thread", fa.numRegs);
  return GPA_OK;
}

template <int D, bool CAUSAL, bool HALVES>
static int launch(const Params& p, const TcPlan& t, cudaStream_t st) {
  static bool checked = false;
  if (!checked) {
    const int rc = check_regs<D, CAUSAL, HALVES>();
    if (rc) return rc;
    checked = true;
  }
  CUtensorMap mq, mkp, mvp, mko, mvo;
  // the folded tokens of all requests are one dim
  const int64_t nreq = t.fold ? 1 : p.requests;
  const int64_t q_tok = p.queries > 1 ? p.q_sm : p.q_sr;
  int rc = make_map(&mq, p.q, D, p.heads, t.tokens, nreq, p.q_sh, t.fold ? q_tok : p.q_sm, p.q_sr, p.group, t.per_tile);
  const bool pre = p.prefix > 0, own = !t.fold && p.cache > 0;
  if (!rc && pre) rc = make_map(&mkp, p.kp, D, p.prefix, p.kv_heads, 1, p.kp_sn, p.kp_sh, 0, TM, 1);
  if (!rc && pre) rc = make_map(&mvp, p.vp, D, p.prefix, p.kv_heads, 1, p.vp_sn, p.vp_sh, 0, TM, 1);
  if (!rc && own) rc = make_map(&mko, p.ko, D, p.cache, p.kv_heads, p.requests, p.ko_sn, p.ko_sh, p.ko_sr, TM, 1);
  if (!rc && own) rc = make_map(&mvo, p.vo, D, p.cache, p.kv_heads, p.requests, p.vo_sn, p.vo_sh, p.vo_sr, TM, 1);
  if (rc) return rc;
  if (!pre) mkp = mko, mvp = mvo;   // never read
  if (!own) mko = mkp, mvo = mvp;
  cudaError_t e = cudaFuncSetAttribute(tc_kernel<D, CAUSAL, HALVES>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcSmem<D, HALVES>::ALLOC);
  if (e != cudaSuccess) return fail(GPA_ERR_CUDA, "gpa_attention_shared_prefix: %s", cudaGetErrorString(e));
  tc_kernel<D, CAUSAL, HALVES><<<t.ctas, TC_THREADS, TcSmem<D, HALVES>::ALLOC, st>>>(mq, mkp, mvp, mko, mvo, p, t);
  return check_launch("gpa_attention_shared_prefix");
}

template <int D>
static int launch_form(const Params& p, const TcPlan& t, cudaStream_t st) {
  const bool causal = p.causal && !t.fold;
  if (t.halves) return causal ? launch<D, true, true>(p, t, st) : launch<D, false, true>(p, t, st);
  return causal ? launch<D, true, false>(p, t, st) : launch<D, false, false>(p, t, st);
}

int launch_tc(const Params& p, int head_dim, const TcPlan& t, cudaStream_t st) {
  return head_dim == 64 ? launch_form<64>(p, t, st) : launch_form<128>(p, t, st);
}

}  // namespace prefix
}  // namespace gpa
