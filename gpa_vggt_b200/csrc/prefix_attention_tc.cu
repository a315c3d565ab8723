// Attention over a shared prefix and own keys for many query rows, on the
// 5th-generation tensor cores (see prefix_attention.cu for the call).
//
// One CTA takes two 128-row tiles of one key/value head and one chunk of the key
// tiles: the prefix's, then the request's own ones, in one online softmax.  384
// threads:
//   warp 0     TMA producer: Q once, then K and V tiles of 128 keys through a
//              ring each; writes a tile's bias / scale as three bf16 terms (24
//              bits) that one more K=16 step adds to the scores, -inf for keys
//              that are out.
//   warps 1-2  MMA issuers, one per row tile: S = Q K^T (+ bias), O += P V with P
//              from TMEM.  Before a tile's first product they zero the K and V
//              rows of keys that are out (past a request's length, or -inf in the
//              bias), whose memory may hold anything.
//   warps 4-11 two softmax warpgroups, a thread per row: S from TMEM, running
//              maximum that moves only by more than 2^8, P back as bf16.
// At head_dim 64 S, P and O of both tiles fit TMEM side by side and S(j+1) runs
// during the softmax of S(j).  At 128 P(j) takes the columns of S(j), and S(j+1)
// waits for O += P(j) V; the other tile's softmax runs meanwhile.
#include "prefix_attention.cuh"

namespace gpa {
namespace prefix {

constexpr int TC_THREADS = 384;
constexpr int TM = 128;   // rows and keys per tile
constexpr int XTILE = TM * 16 * 2;
// Finite biases end here (log2 units).  A row of nothing but the type's lowest
// value spreads evenly: scores up to 64 vanish beside 2^30, and c*x - c*m, off by
// the rounding of c*m (at most 64, the same for all of a row's keys), stays inside
// the exponent's range.
constexpr float kBiasLimit = 1073741824.f;
constexpr int TC_REGS = 168, TC_LOW = 80, TC_HIGH = 208;
static_assert(TC_LOW * 128 + TC_HIGH * 256 <= TC_REGS * TC_THREADS, "register split");

template <int D>
struct TcSmem {
  static constexpr int HALVES = D / 64;          // a row is HALVES swizzled rows of 128 bytes
  static constexpr int HALF = TM * 128;          // 16 KB
  static constexpr int TILE = HALVES * HALF;
  static constexpr int STAGES = D == 64 ? 3 : 2;
  static constexpr int Q = 0;                    // 2 tiles
  static constexpr int K = Q + 2 * TILE;
  static constexpr int V = K + STAGES * TILE;
  static constexpr int ONES = V + STAGES * TILE;
  static constexpr int BETA = ONES + XTILE;
  static constexpr int MASK = BETA + STAGES * XTILE;   // 4 words per stage
  static constexpr int BARS = MASK + STAGES * 16;
  static constexpr int TOTAL = BARS + 256;
  static constexpr int ALLOC = TOTAL + 1024;
  static_assert((1 + 4 * STAGES + 8) * 8 + 8 <= 256, "barrier area");
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

// The two softmax warpgroups.
__device__ __forceinline__ void named_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// 2 of 8 exponentials on the FMA pipe, the rest on MUFU
__device__ __forceinline__ void exp8(const float* x, float* e) {
#pragma unroll
  for (int i = 0; i < 6; ++i) e[i] = fast_exp2(x[i]);
  exp2_poly2<3>(x[6], x[7], e[6], e[7]);
}

template <int D>
__global__ void __launch_bounds__(TC_THREADS, 1)
    tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kp,
              const __grid_constant__ CUtensorMap map_vp, const __grid_constant__ CUtensorMap map_ko,
              const __grid_constant__ CUtensorMap map_vo, const Params p, const TcPlan tc) {
  using SM = TcSmem<D>;
  constexpr int ST = SM::STAGES;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  asm volatile("griddepcontrol.launch_dependents;");   // the join may be launched, and waits for this grid's end

  // the item: row tiles fastest, then requests, so that CTAs running together
  // read the same keys of the prefix
  int it = blockIdx.x;
  const int pair = it % tc.pairs;
  it /= tc.pairs;
  const int nreq = tc.fold ? 1 : p.requests;
  const int req = it % nreq;
  it /= nreq;
  const int split = it % tc.splits;
  const int kh = it / tc.splits;
  const int tok0 = pair * 2 * tc.per_tile;
  const int qlen = tc.fold ? p.queries : query_count(p, req);
  const int tok_end = tc.fold ? tc.tokens : qlen;
  if (tok0 >= tok_end) return;   // padding only: nothing to write
  const int active = tok0 + tc.per_tile < tok_end ? 2 : 1;   // row tiles with rows
  const int len = tc.fold ? 0 : own_length(p, req);
  // with an order, no row of this item sees an own key from here on
  const int own_end = p.causal ? min(len, max(0, len - qlen + min(tok0 + 2 * tc.per_tile, qlen))) : len;
  const int tp = (p.prefix + TM - 1) / TM;
  const int j0 = split * tc.per;
  const int nk = max(0, min(tp + (own_end + TM - 1) / TM, j0 + tc.per) - j0);
  // Two streams of work for the issuers and softmax warpgroups: the two row
  // tiles over the same key tiles, or, where only one has rows, that one over the
  // even and the odd key tiles (joined at the end).
  const bool halves = active == 1 && nk > 1;
  const int streams = nk > 1 ? 2 : active;
  const bool partial = p.s1 + p.s2 > 1;
  auto row_of = [&](int t, int i) {
    Row w;
    const int tl = i / p.group;
    const int tok = tok0 + t * tc.per_tile + tl;
    w.h = kh * p.group + (i - tl * p.group);
    w.live = tl < tc.per_tile && tok < tok_end;
    w.r = req;
    w.m = tok;
    if (tc.fold) {
      w.r = tok / p.queries;
      w.m = tok - w.r * p.queries;
      if (w.live && p.q_len) w.live = w.m < __ldg(p.q_len + w.r);
    }
    return w;
  };
  if (nk == 0) {   // no keys in this chunk
    for (int i = threadIdx.x; i < 2 * TM; i += TC_THREADS) {
      const Row w = row_of(i / TM, i % TM);
      if (!w.live) continue;
      if (partial) {
        p.ws_ml[split * p.rows + row_index(p, w)] = make_float2(-INFINITY, 0.f);
      } else {
        uint4* o = reinterpret_cast<uint4*>(p.o + w.r * p.o_sr + w.h * p.o_sh + w.m * p.o_sm);
        for (int u = 0; u < D / 8; ++u) o[u] = make_uint4(0u, 0u, 0u, 0u);
        if (p.lse) p.lse[w.r * p.lse_sr + w.h * p.lse_sh + w.m] = -INFINITY;
      }
    }
    return;
  }
  // key tile j (of this chunk): the prefix's or an own one
  struct Tile {
    bool own;
    int key0, valid;   // keys of the tile that exist
  };
  auto tile_of = [&](int j) {
    Tile t;
    t.own = j0 + j >= tp;
    t.key0 = (t.own ? j0 + j - tp : j0 + j) * TM;
    t.valid = min(TM, (t.own ? len : p.prefix) - t.key0);
    return t;
  };
  auto has_beta = [&](const Tile& t) { return t.valid < TM || (!t.own && p.bias != nullptr); };

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + SM::BARS);
  uint64_t* k_full = q_full + 1;       // TMA landed
  uint64_t* v_full = k_full + ST;
  uint64_t* k_empty = v_full + ST;
  uint64_t* v_empty = k_empty + ST;
  uint64_t* s_full = v_empty + ST;     // 2
  uint64_t* s_empty = s_full + 2;      // 2
  uint64_t* p_full = s_empty + 2;      // 2
  uint64_t* o_done = p_full + 2;       // 2
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = warp_id(), lane = lane_id();

  if (threadIdx.x == 0) {
    bar_init(q_full, 1);
    for (int s = 0; s < ST; ++s) {
      bar_init(&k_full[s], 1);
      bar_init(&v_full[s], 1);
      bar_init(&k_empty[s], active);   // one arrival per stream that reads the tile
      bar_init(&v_empty[s], active);
    }
    for (int t = 0; t < 2; ++t) {
      bar_init(&s_full[t], 1);
      bar_init(&s_empty[t], 4);
      bar_init(&p_full[t], 4);
      bar_init(&o_done[t], 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tmem_slot;
  auto wait = [&](uint64_t* bar, uint32_t parity) {   // the whole warp, bounded
    return __all_sync(0xffffffffu, wait_bar(bar, parity & 1, abort_flag, p.status, kDevTimeout)) != 0;
  };
  // TMEM columns of a row tile
  auto col_s = [](int t) { return (uint32_t)(t * TM); };
  auto col_o = [](int t) { return (uint32_t)(256 + t * D); };
  auto col_p = [](int t) { return (uint32_t)(D == 64 ? 384 + t * 64 : t * TM); };

  if (warp < 4) {
    regs_dec<TC_LOW>();
    if (warp == 0) {
      // ------------------------------ producer ------------------------------
      if (lane == 0) {
        bar_expect_tx(q_full, active * SM::HALVES * p.group * tc.per_tile * 128);
        for (int t = 0; t < active; ++t)
          for (int h = 0; h < SM::HALVES; ++h)
            tma_load_4d(&map_q, q_full, smem + SM::Q + t * SM::TILE + h * SM::HALF, h * 64, kh * p.group,
                        tok0 + t * tc.per_tile, req);
      }
      uint32_t* w = reinterpret_cast<uint32_t*>(smem + SM::ONES);
      for (int i = lane; i < XTILE * (1 + ST) / 4; i += 32) w[i] = 0u;
      __syncwarp();
      for (int row = lane; row < TM; row += 32)   // 1, 1, 1, 0, ...
        *reinterpret_cast<uint2*>(smem + SM::ONES + xtile_off(row, 0)) = make_uint2(0x3F803F80u, 0x3F80u);
      const float* brow = p.bias ? p.bias + kh * p.bias_sh : nullptr;
      const float inv_scale = 1.0f / p.scale, most = kBiasLimit / p.scale_log2;
      float braw[4];
      auto load_bias = [&](int j) {   // raw bias of a tile, one tile ahead of its use
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = (j0 + j) * TM + i * 32 + lane;
          braw[i] = (brow && j0 + j < tp && key < p.prefix) ? __ldg(brow + key) : 0.f;
        }
      };
      load_bias(0);
      int issued_k = 0, issued_v = 0;
      for (int j = 0; j < nk; ++j) {
        const int s = j % ST;
        const uint32_t ph = (j / ST) & 1;
        const Tile t = tile_of(j);
        if (!wait(&k_empty[s], ph ^ 1)) break;
        if (has_beta(t)) {
          uint32_t* mask = reinterpret_cast<uint32_t*>(smem + SM::MASK + s * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = i * 32 + lane;
            const bool in = row < t.valid && braw[i] > -INFINITY;   // NaN takes a key out too
            const float beta = in ? fminf(fmaxf(braw[i] * inv_scale, -most), most) : -INFINITY;
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
            if (lane == 0) mask[i] = out;
          }
          fence_async_smem();
          __syncwarp();
        }
        load_bias(j + 1);
        if (lane == 0) {
          bar_expect_tx(&k_full[s], SM::TILE);
          for (int h = 0; h < SM::HALVES; ++h)
            tma_load_4d(t.own ? &map_ko : &map_kp, &k_full[s], smem + SM::K + s * SM::TILE + h * SM::HALF, h * 64,
                        t.key0, kh, t.own ? req : 0);
        }
        issued_k = j + 1;
        if (!wait(&v_empty[s], ph ^ 1)) break;
        if (lane == 0) {
          bar_expect_tx(&v_full[s], SM::TILE);
          for (int h = 0; h < SM::HALVES; ++h)
            tma_load_4d(t.own ? &map_vo : &map_vp, &v_full[s], smem + SM::V + s * SM::TILE + h * SM::HALF, h * 64,
                        t.key0, kh, t.own ? req : 0);
        }
        issued_v = j + 1;
      }
      if (lane == 0) {   // copies in flight land before the CTA exits
        const unsigned long long t0 = global_ns();
        drain_bar(q_full, 0, t0);
        for (int j = max(0, issued_k - ST); j < issued_k; ++j) drain_bar(&k_full[j % ST], (j / ST) & 1, t0);
        for (int j = max(0, issued_v - ST); j < issued_v; ++j) drain_bar(&v_full[j % ST], (j / ST) & 1, t0);
      }
    } else if (warp - 1 < streams) {
      // ------------------------------ MMA issuers ------------------------------
      // j counts this stream's key tiles, key_tile(j) the chunk's
      const int t = warp - 1;
      const int n = halves ? (nk - t + 1) >> 1 : nk;
      auto key_tile = [&](int j) { return halves ? 2 * j + t : j; };
      const bool leader = elect_one();
      constexpr uint32_t idesc_s = idesc_bf16(TM, TM, false, false);
      constexpr uint32_t idesc_o = idesc_bf16(TM, D, false, true);
      const uint64_t dQ = sdesc_sw128(smem_u32(smem + SM::Q + (halves ? 0 : t) * SM::TILE), 16, 1024);
      const uint64_t dK = sdesc_sw128(smem_u32(smem + SM::K), 16, 1024);
      const uint64_t dV = sdesc_sw128(smem_u32(smem + SM::V), SM::HALF, 1024);
      const uint64_t dOnes = sdesc_plain(smem_u32(smem + SM::ONES));
      const uint64_t dBeta = sdesc_plain(smem_u32(smem + SM::BETA));
      const uint32_t dS = tbase + col_s(t), dO = tbase + col_o(t), dP = tbase + col_p(t);
      auto issue_s = [&](int j) {
        const int jt = key_tile(j), st = jt % ST;
        const bool beta = has_beta(tile_of(jt));
        if (leader) {
          const uint64_t bk = dK + (uint64_t)(st * (SM::TILE >> 4));
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint64_t off = (uint64_t)((k >> 2) * (SM::HALF >> 4) + (k & 3) * 2);
            umma_bf16(dS, dQ + off, bk + off, idesc_s, k != 0);
          }
          if (beta) umma_bf16(dS, dOnes, dBeta + (uint64_t)(st * (XTILE >> 4)), idesc_s, 1);
          umma_commit(&s_full[t]);
          umma_commit(&k_empty[st]);
        }
        __syncwarp();
      };
      auto issue_o = [&](int j) {
        const int st = key_tile(j) % ST;
        if (leader) {
          const uint64_t bv = dV + (uint64_t)(st * (SM::TILE >> 4));
#pragma unroll
          for (int ks = 0; ks < TM / 16; ++ks)
            umma_bf16_ts(dO, dP + ks * 8, bv + (uint64_t)(ks * (2048 >> 4)), idesc_o, (j > 0 || ks > 0));
          umma_commit(&o_done[t]);
          umma_commit(&v_empty[st]);
        }
        __syncwarp();
      };
      // The rows to zero of a key tile, read once its K has landed (the producer
      // reuses the words before its V is used).
      auto rows_out = [&](int j) {
        const Tile kt = tile_of(key_tile(j));
        return (kt.own ? kt.valid < TM : p.bias != nullptr)
                   ? *reinterpret_cast<const uint4*>(smem + SM::MASK + (key_tile(j) % ST) * 16)
                   : make_uint4(0u, 0u, 0u, 0u);
      };
      // Where both issuers read a tile, the second writes the same zeros.
      auto zero_rows = [&](const uint4& m, int base, int j) {
        if (!(m.x | m.y | m.z | m.w)) return;
        uint8_t* tile = smem + base + (key_tile(j) % ST) * SM::TILE + (lane >> 3) * SM::HALF + (lane & 7) * 16;
        for (int row = 0; row < TM; ++row) {
          const uint32_t word = row < 64 ? (row < 32 ? m.x : m.y) : (row < 96 ? m.z : m.w);
          if ((word >> (row & 31) & 1) && lane < 8 * SM::HALVES)
            *reinterpret_cast<uint4*>(tile + row * 128) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_async_smem();
        __syncwarp();
      };
      auto wait_tile = [&](uint64_t* bar, int j) { return wait(&bar[key_tile(j) % ST], key_tile(j) / ST); };
      uint4 out_now = make_uint4(0u, 0u, 0u, 0u), out_next = out_now;
      auto scores = [&](int j) {   // once K has landed
        tc_fence_after();
        out_next = rows_out(j);
        zero_rows(out_next, SM::K, j);
        issue_s(j);
      };
      bool okw = wait(q_full, 0) && wait_tile(k_full, 0);
      if (okw) scores(0);
      for (int j = 0; okw && j < n; ++j) {
        out_now = out_next;
        if (D == 64 && j + 1 < n) {
          okw = wait(&s_empty[t], j) && wait_tile(k_full, j + 1);
          if (!okw) break;
          scores(j + 1);
        }
        okw = wait(&p_full[t], j) && wait_tile(v_full, j);
        if (!okw) break;
        tc_fence_after();
        zero_rows(out_now, SM::V, j);
        issue_o(j);
        if (D == 128 && j + 1 < n) {
          // S(j+1) overwrites P(j), which O += P(j) V still reads until it is done
          okw = wait_tile(k_full, j + 1) && wait(&o_done[t], j);
          if (!okw) break;
          scores(j + 1);
        }
      }
    }
  } else {
    regs_inc<TC_HIGH>();
    // ------------------------------ softmax ------------------------------
    const int t = (warp - 4) >> 2;
    if (t < streams) {
      const int n = halves ? (nk - t + 1) >> 1 : nk;
      const int quad = warp & 3;
      const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
      const uint32_t tS = tbase + lane_off + col_s(t), tO = tbase + lane_off + col_o(t), tP = tbase + lane_off + col_p(t);
      const Row row = row_of(halves ? 0 : t, quad * 32 + lane);
      const bool idle = !__any_sync(0xffffffffu, row.live);   // a warp without rows only keeps the barriers going
      // own keys that this row sees end here
      const bool ordered = p.causal && !tc.fold;
      const int limit = ordered ? len - qlen + row.m + 1 : 0x7fffffff;
      constexpr float kNoMax = -3.0e38f;   // no key yet
      float m_raw = kNoMax, l = 0.f;       // running maximum (score units), row sum
      float neg_mc = 0.f;                  // -c2 * m_raw
      const float c2 = p.scale_log2;
      bool okw = true;
      auto quarter = [&](float* xq, float neg_mc, float* acc, uint32_t* pk) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float* xg = xq + g * 8;
#pragma unroll
          for (int i = 0; i < 8; i += 2) ffma2(xg[i], xg[i + 1], xg[i], xg[i + 1], c2, c2, neg_mc, neg_mc);
          float e[8];
          exp8(xg, e);
#pragma unroll
          for (int i = 0; i < 8; i += 2) fadd2(acc[i], acc[i + 1], acc[i], acc[i + 1], e[i], e[i + 1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) pk[g * 4 + i] = pack_bf16x2(e[2 * i], e[2 * i + 1]);
        }
      };
      if (idle) {
        for (int j = 0; j < n; ++j) {
          // S(j+1) may be there before the other warps' P(j): no second arrival in one phase
          okw = wait(&s_full[t], j) && (j == 0 || wait(&p_full[t], j - 1));
          if (!okw) break;
          if (lane == 0) {
            if (D == 64) bar_arrive(&s_empty[t]);
            bar_arrive(&p_full[t]);
          }
        }
      }
      for (int j = idle ? n : 0; j < n; ++j) {
        if (!wait(&s_full[t], j)) { okw = false; break; }
        tc_fence_after();
        float x[TM];
#pragma unroll
        for (int c = 0; c < TM / 32; ++c) tmem_ld32f(tS + c * 32, x + c * 32);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (D == 64 && lane == 0) bar_arrive(&s_empty[t]);
        if (ordered) {   // keys ahead of this row
          const Tile kt = tile_of(halves ? 2 * j + t : j);
          if (kt.own && __any_sync(0xffffffffu, limit < kt.key0 + TM)) {
            const int end = limit - kt.key0;
#pragma unroll
            for (int c = 0; c < TM; ++c)
              if (c >= end) x[c] = -INFINITY;
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < TM / 4; ++c) {
          mx[c & 3] = max3_nan(mx[c & 3], x[4 * c + 0], x[4 * c + 1]);
          mx[c & 3] = max3_nan(mx[c & 3], x[4 * c + 2], x[4 * c + 3]);
        }
        const float mt = max3_nan(max3_nan(mx[0], mx[0], mx[1]), mx[2], mx[3]);
        float alpha = 1.f;
        // the maximum moves: also the first time, and for a NaN (never for a row without keys)
        const bool moved = row.live && !((mt - m_raw) * c2 <= 8.0f);
        const bool any_moved = __any_sync(0xffffffffu, moved);
        if (any_moved) {
          if (moved) {
            alpha = fast_exp2((m_raw - mt) * c2);
            l = mt < INFINITY ? l * alpha : NAN;   // a NaN or infinite score: the row is NaN (the polynomial would lose it)
            m_raw = mt < INFINITY ? mt : 0.f;
            neg_mc = -m_raw * c2;
          }
        }
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        uint32_t pk[4][16];
#pragma unroll
        for (int qt = 0; qt < 4; ++qt) {
          quarter(x + qt * 32, neg_mc, acc, pk[qt]);
          if (D == 128) {   // S(j) came after O += P(j-1) V
            tmem_st16(tP + qt * 16, pk[qt]);
          } else if (qt == 1) {
            if (j > 0) {    // P and O are busy until O += P(j-1) V is done
              if (!wait(&o_done[t], j - 1)) { okw = false; break; }
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
          for (int c = 0; c < D / 32; ++c) {
            tmem_ld32(tO + c * 32, ov);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
            tmem_st32(tO + c * 32, ov);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&p_full[t]);
      }
      if (okw) okw = wait(&o_done[t], n - 1);
      tc_fence_after();
      // The second half's output goes through the rings' memory (all of it has
      // been read once both halves are done), feature-major: a thread per row.
      float* xo = reinterpret_cast<float*>(smem + SM::K) + quad * 32 + lane;
      float* xml = reinterpret_cast<float*>(smem + SM::Q) + (quad * 32 + lane) * 2;
      float f1 = 0.f;
      if (halves) {
        named_sync();
        if (t == 1 && okw) {
          xml[0] = m_raw;
          xml[1] = l;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t ov[32];
            tmem_ld32(tO + c * 32, ov);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) xo[(c * 32 + i) * TM] = __uint_as_float(ov[i]);
          }
        }
        named_sync();
      }
      if (okw && !*abort_flag && !(halves && t == 1)) {
        float f0 = 1.f;
        if (halves) {
          const float m1 = xml[0], m = fmaxf(m_raw, m1);
          f0 = fast_exp2((m_raw - m) * c2);
          f1 = fast_exp2((m1 - m) * c2);
          l = l * f0 + xml[1] * f1;
          m_raw = m;
        }
        const bool some = m_raw > kNoMax;   // else the sum holds the polynomial's 2^-126
        const float inv = some ? 1.0f / l : 0.f;
        const int64_t at = split * p.rows + row_index(p, row);
        __nv_bfloat16* orow = p.o + row.r * p.o_sr + row.h * p.o_sh + row.m * p.o_sm;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t ov[32];
          tmem_ld32(tO + c * 32, ov);
          tmem_wait_ld();
          if (!row.live) continue;
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(ov[i]);
          if (halves) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = fmaf(v[i], f0, xo[(c * 32 + i) * TM] * f1);
          }
          if (partial) {
            float4* w = reinterpret_cast<float4*>(p.ws_o + at * D + c * 32);
#pragma unroll
            for (int u = 0; u < 8; ++u) w[u] = make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
          } else {
            uint32_t w[16];
#pragma unroll
            for (int u = 0; u < 16; ++u) w[u] = some ? pack_bf16x2(v[2 * u] * inv, v[2 * u + 1] * inv) : 0u;
#pragma unroll
            for (int u = 0; u < 4; ++u)
              reinterpret_cast<uint4*>(orow + c * 32)[u] = make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
          }
        }
        if (row.live) {
          if (partial)
            p.ws_ml[at] = some ? make_float2(m_raw * c2, l) : make_float2(-INFINITY, 0.f);
          else if (p.lse)
            p.lse[row.r * p.lse_sr + row.h * p.lse_sh + row.m] = some ? m_raw * c2 + log2f(l) : -INFINITY;
        }
      }
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
  if (!(p.scale > 1e-6f && p.scale < 1e6f) || p.group > TM) return false;
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
template <int D>
static int check_regs() {
  cudaFuncAttributes fa;
  if (cudaFuncGetAttributes(&fa, tc_kernel<D>) != cudaSuccess)
    return fail(GPA_ERR_CUDA, "gpa_attention_shared_prefix: cudaFuncGetAttributes failed");
  if (fa.numRegs * TC_THREADS < TC_LOW * 128 + TC_HIGH * 256)
    return fail(GPA_ERR_CUDA, "gpa_attention_shared_prefix: kernel built with %d registers/thread", fa.numRegs);
  return GPA_OK;
}

template <int D>
static int launch(const Params& p, const TcPlan& t, cudaStream_t st) {
  static bool checked = false;
  if (!checked) {
    const int rc = check_regs<D>();
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
  cudaError_t e = cudaFuncSetAttribute(tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcSmem<D>::ALLOC);
  if (e != cudaSuccess) return fail(GPA_ERR_CUDA, "gpa_attention_shared_prefix: %s", cudaGetErrorString(e));
  const int64_t items = (int64_t)t.pairs * nreq * t.splits * p.kv_heads;
  tc_kernel<D><<<(unsigned)items, TC_THREADS, TcSmem<D>::ALLOC, st>>>(mq, mkp, mvp, mko, mvo, p, t);
  return check_launch("gpa_attention_shared_prefix");
}

int launch_tc(const Params& p, int head_dim, const TcPlan& t, cudaStream_t st) {
  return head_dim == 64 ? launch<64>(p, t, st) : launch<128>(p, t, st);
}

}  // namespace prefix
}  // namespace gpa
