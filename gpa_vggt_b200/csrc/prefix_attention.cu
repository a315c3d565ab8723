// Attention of a batch of requests over prefix keys that all of them share and
// over each request's own cached keys (one softmax over both):
//   s_ij = scale * q_i . k_j + bias_j     (prefix keys; own keys without bias)
//   o_i  = sum_j softmax_j(s_i) v_j,      lse_i = log2 of the softmax denominator
//
// The prefix is read once for all requests: the queries of every request that
// use one key/value head are rows of the same tile.  The keys are split into
// chunks, an item is (row tile, key/value head, chunk) of the prefix or of one
// request's cache, and each writes its unnormalised output, maximum and sum; a
// second kernel joins the chunks of a row:
//   m = max m_c, l = sum l_c 2^(m_c - m), o = sum o_c 2^(m_c - m) / l.
// Scores, statistics and partial outputs are fp32; the probabilities are rounded
// to bf16 for the product with V (their sum is not).
//
// This file: few rows per tile (one token, or a few, of each request), 16 to 64
// rows on mma.sync tiles.  Up to 16 rows a call is a stream of K and V from HBM: 5
// streams of one token over 219,840 + 2,748 keys of 16 heads read 0.94 GB in 143 us
// (6.57 TB/s).  From 32 rows on the tensor unit bounds it, which ends at 0.2-0.25
// PFLOP/s for mma.sync (with the join, 16, 32 and 64 rows over 66,845 keys of 16
// heads: 55, 62 and 95 us).  K and V come through a cp.async ring of three 64-key
// tiles, with two to four CTAs per SM: 64 KB and more of loads in flight, and enough
// warps that one's exponentials run beside another's products.  Many rows:
// prefix_attention_tc.cu.
#include <type_traits>

#include "prefix_attention.cuh"

namespace gpa {
namespace prefix {

constexpr int BN = 64;         // keys per tile
constexpr int THREADS = 128;
constexpr int kSlotTiles = 2;  // at least this many tiles per chunk (2 requests, 2,361 + 100 keys: 8.3 us; 4: 8.9)
constexpr int kSms = 148;
constexpr int kJoinCtas = kSms * 8;   // the most CTAs of join_tiles_kernel with 8 features a thread
constexpr int kLeastSteps = 4;  // the tensor-core kernel cuts no item into parts of fewer steps

// CTAs per SM for row tiles of 16 * wm1 rows over the prefix and 16 * wm2 over the
// caches.  At head_dim 64 four with a ring of three tiles hide more of the loads and
// of each other's exponentials than three with one of four (5 streams over 219,840 +
// 2,748 keys 143 us, 147; 64 over 66,845 + 1,374 113, 116), but 32-row tiles, and
// higher ones over the caches, need more than the 128 registers that leaves (32 rows
// over 66,845 keys: 62 us with three, 66 with four; 8 x 64 tokens over 2,000 32, 34).
constexpr int resident(int head_dim, int wm1, int wm2) { return head_dim == 128 ? 2 : wm2 == 1 && wm1 != 2 ? 4 : 3; }

template <int D>
struct Cfg {
  static constexpr int STAGES = 3;
  static constexpr int TILE = BN * D * 2;                    // bytes of a K or V tile
  static constexpr int STAGE = 2 * TILE + BN * 4;            // K, V, bias
  static constexpr int SMEM = STAGES * STAGE;
  static constexpr int CTAS = D == 64 ? 4 : 2;               // resident at most
  static_assert(SMEM * CTAS <= 227 * 1024 - CTAS * 1024, "shared memory of the resident CTAs");
  static_assert(4 * 16 * (D + 2) * 4 <= SMEM, "the warps' partial outputs reuse the ring");
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
  const int n = in ? 16 : 0;   // zero fill past the end
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Byte offset of 16-byte chunk c of key row in a tile: rows of D bf16, the
// chunk's low three bits swapped around by the row, so that eight rows of one
// chunk column lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t swz(int row, int c) {
  return row * (D * 2) + (((c & ~7) | ((c ^ row) & 7)) << 4);
}

// A prefix bias in log2 units.  -inf (or NaN) takes the key out; the type's
// lowest values stay finite, so keys that all carry them are still weighed.
__device__ __forceinline__ float bias_log2(float b) {
  return b > -INFINITY ? fminf(fmaxf(b, -kBiasLimit), kBiasLimit) * 1.4426950408889634f : -INFINITY;
}

// Tokens are counted through all requests (prefix) or within one (own).
template <bool OWN>
__device__ __forceinline__ Row row_of(const Params& p, int i, int req, int kh) {
  Row w;
  const int tok = i / p.group;
  w.h = kh * p.group + (i - tok * p.group);
  w.r = OWN ? req : tok / p.queries;
  w.m = OWN ? tok : tok - w.r * p.queries;
  w.live = OWN ? tok < p.queries : w.r < p.requests;
  if (w.live && p.q_len) w.live = w.m < __ldg(p.q_len + w.r);
  return w;
}

// One item.  WM warps of 16 rows each; the 4 / WM warps that share the rows
// split each tile's keys and are joined at the end.
template <int D, int WM, bool OWN>
__device__ __forceinline__ void run_item(const Params& p, uint8_t* smem, int kh, int req, int tile, int slot) {
  using C = Cfg<D>;
  constexpr int WK = 4 / WM;
  constexpr int KW = BN / WK;          // keys of a tile per warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wm = warp % WM, wk = warp / WM;
  const int row0 = tile * (16 * WM) + wm * 16;

  const int len = OWN ? own_length(p, req) : p.prefix;
  const int qlen = OWN ? query_count(p, req) : p.queries;
  const int k0 = slot * p.chunk, k1 = min(len, k0 + p.chunk);
  const int64_t base = (int64_t)(OWN ? p.s1 + slot : slot) * p.rows;
  auto row_at = [&](const Row& w) { return base + row_index(p, w); };
  if (k0 >= k1) {   // nothing here: no output, a sum of zero
    if (threadIdx.x < 16 * WM) {
      const Row w = row_of<OWN>(p, tile * (16 * WM) + threadIdx.x, req, kh);
      if (w.live) p.ws_ml[row_at(w)] = make_float2(-INFINITY, 0.f);
    }
    return;
  }
  const Row ra = row_of<OWN>(p, row0 + (lane >> 2), req, kh), rb = row_of<OWN>(p, row0 + (lane >> 2) + 8, req, kh);
  const int nt = (k1 - k0 + BN - 1) / BN;
  // keys that a row sees end here (own keys in order: the last query sees them all)
  const int ea = OWN && p.causal ? len - qlen + ra.m + 1 : k1, eb = OWN && p.causal ? len - qlen + rb.m + 1 : k1;

  const __nv_bfloat16* kbase = OWN ? p.ko + req * p.ko_sr + kh * p.ko_sh : p.kp + kh * p.kp_sh;
  const __nv_bfloat16* vbase = OWN ? p.vo + req * p.vo_sr + kh * p.vo_sh : p.vp + kh * p.vp_sh;
  const int64_t ksn = OWN ? p.ko_sn : p.kp_sn, vsn = OWN ? p.vo_sn : p.vp_sn;
  const float* bias = OWN || !p.bias ? nullptr : p.bias + kh * p.bias_sh;
  const uint32_t sbase = smem_u32(smem);

  auto issue = [&](int j) {
    if (j < nt) {
      const uint32_t st = sbase + (j % C::STAGES) * C::STAGE;
      constexpr int CPR = D / 8;                       // 16-byte chunks per row
      const int c = threadIdx.x % CPR;
#pragma unroll
      for (int i = 0; i < BN / (THREADS / CPR); ++i) {
        const int row = threadIdx.x / CPR + i * (THREADS / CPR);
        const int key = k0 + j * BN + row;
        const bool in = key < k1;
        const int64_t kk = in ? key : k0;
        cp16(st + swz<D>(row, c), kbase + kk * ksn + c * 8, in);
        cp16(st + C::TILE + swz<D>(row, c), vbase + kk * vsn + c * 8, in);
      }
      if (bias && threadIdx.x < BN) {
        const int key = min(k0 + j * BN + (int)threadIdx.x, k1 - 1);
        cp4(st + 2 * C::TILE + threadIdx.x * 4, bias + key);
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int j = 0; j < C::STAGES - 1; ++j) issue(j);

  // Q fragments straight from memory: 16 rows x D of this warp
  uint32_t qf[D / 16][4];
  {
    const __nv_bfloat16* qa = p.q + ra.r * p.q_sr + ra.h * p.q_sh + ra.m * p.q_sm + (lane & 3) * 2;
    const __nv_bfloat16* qb = p.q + rb.r * p.q_sr + rb.h * p.q_sh + rb.m * p.q_sm + (lane & 3) * 2;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      qf[k][0] = ra.live ? __ldg(reinterpret_cast<const uint32_t*>(qa + k * 16)) : 0u;
      qf[k][1] = rb.live ? __ldg(reinterpret_cast<const uint32_t*>(qb + k * 16)) : 0u;
      qf[k][2] = ra.live ? __ldg(reinterpret_cast<const uint32_t*>(qa + k * 16 + 8)) : 0u;
      qf[k][3] = rb.live ? __ldg(reinterpret_cast<const uint32_t*>(qb + k * 16 + 8)) : 0u;
    }
  }
  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float ma = -INFINITY, mb = -INFINITY, la = 0.f, lb = 0.f;

  for (int j = 0; j < nt; ++j) {
    cp_wait<C::STAGES - 2>();
    __syncthreads();
    issue(j + C::STAGES - 1);
    const int st = (j % C::STAGES) * C::STAGE;
    const uint32_t sk = sbase + st, sv = sk + C::TILE;
    float* sb = reinterpret_cast<float*>(smem + st + 2 * C::TILE);
    const int kt = k0 + j * BN;           // first key of the tile
    if (bias) {
      // Keys that the bias takes out count as absent: their K and V may hold
      // anything, so they are zeroed here by every warp that reads them.
      bool out = false;
#pragma unroll
      for (int i = 0; i < KW; i += 32) out |= (KW >= 32 || lane < KW) && !(sb[wk * KW + (i + lane) % KW] > -INFINITY);
      unsigned any = __ballot_sync(0xffffffffu, out);
      if (any) {
        for (int row = wk * KW; row < wk * KW + KW; ++row)
          if (!(sb[row] > -INFINITY) && lane < D / 8) {
            *reinterpret_cast<uint4*>(smem + st + swz<D>(row, lane)) = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(smem + st + C::TILE + swz<D>(row, lane)) = make_uint4(0u, 0u, 0u, 0u);
          }
        __syncwarp();
      }
    }
    float s[KW / 8][4];
#pragma unroll
    for (int n = 0; n < KW / 8; ++n) {
      s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {   // 8 keys x 32 features
        uint32_t b[4];
        ldsm4(sk + swz<D>(wk * KW + n * 8 + (lane & 7), k * 4 + (lane >> 3)), b);
        mma(s[n], qf[2 * k], b[0], b[1]);
        mma(s[n], qf[2 * k + 1], b[2], b[3]);
      }
    }
    // scale, bias, mask
    const bool edge = kt + BN > k1 || (OWN && p.causal && kt + BN > len - qlen + 1);
    float xa = -INFINITY, xb = -INFINITY;
#pragma unroll
    for (int n = 0; n < KW / 8; ++n) {
      const int col = wk * KW + n * 8 + (lane & 3) * 2;
      float b0 = 0.f, b1 = 0.f;
      if (bias) {
        const float2 bb = *reinterpret_cast<const float2*>(sb + col);
        b0 = bias_log2(bb.x);
        b1 = bias_log2(bb.y);
      }
      s[n][0] = fmaf(s[n][0], p.scale_log2, b0);
      s[n][1] = fmaf(s[n][1], p.scale_log2, b1);
      s[n][2] = fmaf(s[n][2], p.scale_log2, b0);
      s[n][3] = fmaf(s[n][3], p.scale_log2, b1);
      if (edge) {
        const int key = kt + col;
        const int ca = min(ea, k1), cb = min(eb, k1);
        if (key >= ca) s[n][0] = -INFINITY;
        if (key + 1 >= ca) s[n][1] = -INFINITY;
        if (key >= cb) s[n][2] = -INFINITY;
        if (key + 1 >= cb) s[n][3] = -INFINITY;
      }
      xa = fmaxf(xa, fmaxf(s[n][0], s[n][1]));
      xb = fmaxf(xb, fmaxf(s[n][2], s[n][3]));
    }
    xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, 1));
    xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, 2));
    xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, 1));
    xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, 2));
    if (xa > ma || xb > mb) {   // quads move on their own
      const float na = fmaxf(ma, xa), nb = fmaxf(mb, xb);
      const float fa = na > ma ? fast_exp2(ma - na) : 1.f, fb = nb > mb ? fast_exp2(mb - nb) : 1.f;
      ma = na;
      mb = nb;
      la *= fa;
      lb *= fb;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][0] *= fa;
        o[i][1] *= fa;
        o[i][2] *= fb;
        o[i][3] *= fb;
      }
    }
    __syncwarp();
    const float sa = ma > -INFINITY ? ma : 0.f, sbm = mb > -INFINITY ? mb : 0.f;
#pragma unroll
    for (int k = 0; k < KW / 16; ++k) {
      uint32_t pf[4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float* x = s[2 * k + u];
        const float e0 = fast_exp2(x[0] - sa), e1 = fast_exp2(x[1] - sa);
        const float e2 = fast_exp2(x[2] - sbm), e3 = fast_exp2(x[3] - sbm);
        la += e0 + e1;
        lb += e2 + e3;
        pf[2 * u] = pack_bf16x2(e0, e1);
        pf[2 * u + 1] = pack_bf16x2(e2, e3);
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {   // 16 keys x 16 features of V
        uint32_t b[4];
        ldsm4t(sv + swz<D>(wk * KW + k * 16 + (lane & 15), d * 2 + (lane >> 4)), b);
        mma(o[2 * d], pf, b[0], b[1]);
        mma(o[2 * d + 1], pf, b[2], b[3]);
      }
    }
  }
  la += __shfl_xor_sync(0xffffffffu, la, 1);
  la += __shfl_xor_sync(0xffffffffu, la, 2);
  lb += __shfl_xor_sync(0xffffffffu, lb, 1);
  lb += __shfl_xor_sync(0xffffffffu, lb, 2);

  if constexpr (WK == 1) {
    if (ra.live) {
      const int64_t at = row_at(ra);
      if ((lane & 3) == 0) p.ws_ml[at] = make_float2(ma, la);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          *reinterpret_cast<float2*>(p.ws_o + at * D + i * 8 + (lane & 3) * 2) = make_float2(o[i][0], o[i][1]);
    }
    if (rb.live) {
      const int64_t at = row_at(rb);
      if ((lane & 3) == 0) p.ws_ml[at] = make_float2(mb, lb);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          *reinterpret_cast<float2*>(p.ws_o + at * D + i * 8 + (lane & 3) * 2) = make_float2(o[i][2], o[i][3]);
    }
  } else {
    // join the WK warps of a row through the ring's memory
    cp_wait<0>();
    __syncthreads();
    float* po = reinterpret_cast<float*>(smem);                 // [4 warps][16 rows][D]
    float2* pm = reinterpret_cast<float2*>(po + 4 * 16 * D);     // [4 warps][16 rows]
    const int a = lane >> 2;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      *reinterpret_cast<float2*>(po + (warp * 16 + a) * D + i * 8 + (lane & 3) * 2) = make_float2(o[i][0], o[i][1]);
      *reinterpret_cast<float2*>(po + (warp * 16 + a + 8) * D + i * 8 + (lane & 3) * 2) = make_float2(o[i][2], o[i][3]);
    }
    if ((lane & 3) == 0) {
      pm[warp * 16 + a] = make_float2(ma, la);
      pm[warp * 16 + a + 8] = make_float2(mb, lb);
    }
    __syncthreads();
    // a warp takes rows in turn, its lanes the features
    for (int i = warp; i < 16 * WM; i += 4) {
      const Row w = row_of<OWN>(p, tile * (16 * WM) + i, req, kh);
      if (!w.live) continue;
      const int q0 = (i >> 4) * 16 + (i & 15);    // this row in the first of its warps
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int c = 0; c < WK; ++c) m = fmaxf(m, pm[c * WM * 16 + q0].x);
      float v[D / 32];
#pragma unroll
      for (int u = 0; u < D / 32; ++u) v[u] = 0.f;
#pragma unroll
      for (int c = 0; c < WK; ++c) {
        const float2 ml = pm[c * WM * 16 + q0];
        const float f = ml.x > -INFINITY ? fast_exp2(ml.x - m) : 0.f;
        l += ml.y * f;
#pragma unroll
        for (int u = 0; u < D / 32; ++u) v[u] = fmaf(f, po[(c * WM * 16 + q0) * D + u * 32 + lane], v[u]);
      }
      const int64_t at = row_at(w);
      if (lane == 0) p.ws_ml[at] = make_float2(m, l);
#pragma unroll
      for (int u = 0; u < D / 32; ++u) p.ws_o[at * D + u * 32 + lane] = v[u];
    }
  }
}

template <int D, int WM1, int WM2>
__global__ void __launch_bounds__(THREADS, resident(D, WM1, WM2)) rows_kernel(const Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  asm volatile("griddepcontrol.launch_dependents;");   // the join may be launched, and waits for this grid's end
  // items of the prefix: row tile fastest (its CTAs share the keys in L2)
  int64_t it = blockIdx.x;
  const int64_t n1 = (int64_t)p.kv_heads * p.s1 * p.rt1;
  if (it < n1) {
    const int t = (int)(it % p.rt1);
    it /= p.rt1;
    run_item<D, WM1, false>(p, smem, (int)(it / p.s1), 0, t, (int)(it % p.s1));
  } else {
    it -= n1;
    const int t = (int)(it % p.rt2);
    it /= p.rt2;
    const int s = (int)(it % p.s2);
    it /= p.s2;
    run_item<D, WM2, true>(p, smem, (int)(it % p.kv_heads), (int)(it / p.kv_heads), t, s);
  }
  // Behind tc_kernel this grid starts before that one's end (neither reads what
  // the other writes); its own end, which the join waits for, must not come first.
  if (blockIdx.x == gridDim.x - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Joins the chunks of a row with W warps (1: a warp's own row, else the block's,
// which take the chunks in turn and are joined like chunks themselves).
template <int D, int W>
__device__ __forceinline__ void join_row(const Params& p, int64_t row, float (*part)[D], float2* part_ml) {
  constexpr int F = D / 32;   // features per lane
  constexpr int U = 8;        // loads in flight
  const int warp = W == 1 ? 0 : threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = (int)((uint32_t)row % (uint32_t)p.heads), tok = (int)((uint32_t)row / (uint32_t)p.heads);
  const int m = (int)((uint32_t)tok % (uint32_t)p.queries), r = (int)((uint32_t)tok / (uint32_t)p.queries);
  const int slots = (p.s1 + p.s2 - warp + W - 1) / W;   // this warp's: warp, warp + W, ...
  const int64_t step = W * p.rows;
  const float2* mlr = p.ws_ml + warp * p.rows + row;
  const float2 first = lane < slots ? mlr[lane * step] : make_float2(-INFINITY, 0.f);
  float mx = first.x;
  for (int s = lane + 32; s < slots; s += 32) mx = fmaxf(mx, mlr[s * step].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  float l = 0.f, v[F];
#pragma unroll
  for (int u = 0; u < F; ++u) v[u] = 0.f;
  const float* orow = p.ws_o + (warp * p.rows + row) * D + lane * F;
  for (int s0 = 0; s0 < slots; s0 += 32) {
    const float2 ml = s0 == 0 ? first : (s0 + lane < slots ? mlr[(s0 + lane) * step] : make_float2(-INFINITY, 0.f));
    const float f = ml.x > -INFINITY ? exp2f(ml.x - mx) : 0.f;
    l = fmaf(ml.y, f, l);
    const int n = min(32, slots - s0);
    for (int i0 = 0; i0 < n; i0 += U) {
      float x[U][F], w[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int s = i0 + i;
        w[i] = __shfl_sync(0xffffffffu, f, s & 31);
        if (s >= n) w[i] = 0.f;
        const float* src = orow + (s0 + s) * step * D;
        if (w[i] > 0.f) {   // an empty chunk wrote no output
          if constexpr (F == 2) {
            const float2 t = *reinterpret_cast<const float2*>(src);
            x[i][0] = t.x; x[i][1] = t.y;
          } else {
            const float4 t = *reinterpret_cast<const float4*>(src);
            x[i][0] = t.x; x[i][1] = t.y; x[i][2] = t.z; x[i][3] = t.w;
          }
        } else {
#pragma unroll
          for (int u = 0; u < F; ++u) x[i][u] = 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int u = 0; u < F; ++u) v[u] = fmaf(w[i], x[i][u], v[u]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if constexpr (W > 1) {
#pragma unroll
    for (int u = 0; u < F; ++u) part[warp][lane * F + u] = v[u];
    if (lane == 0) part_ml[warp] = make_float2(mx, l);
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int i = 0; i < W; ++i) mx = fmaxf(mx, part_ml[i].x);
    l = 0.f;
#pragma unroll
    for (int u = 0; u < F; ++u) v[u] = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float2 ml = part_ml[i];
      const float f = ml.x > -INFINITY ? exp2f(ml.x - mx) : 0.f;
      l = fmaf(ml.y, f, l);
#pragma unroll
      for (int u = 0; u < F; ++u) v[u] = fmaf(f, part[i][lane * F + u], v[u]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;   // no key: zero (a NaN stays one)
  __nv_bfloat16* dst = p.o + r * p.o_sr + h * p.o_sh + m * p.o_sm + lane * F;
  if constexpr (F == 2) {
    *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(v[0] * inv, v[1] * inv);
  } else {
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv));
  }
  if (p.lse && lane == 0) p.lse[r * p.lse_sr + h * p.lse_sh + m] = l == 0.f ? -INFINITY : mx + log2f(l);
}

// Whether a row's chunks are to be joined: not past its request's queries.
__device__ __forceinline__ bool to_join(const Params& p, int64_t row) {
  if (row >= p.rows) return false;
  if (!p.q_len) return true;
  const uint32_t tok = (uint32_t)row / (uint32_t)p.heads;
  return (int)(tok % (uint32_t)p.queries) < __ldg(p.q_len + tok / (uint32_t)p.queries);
}

// Joins rows_kernel's chunks, a row with W warps (1, or a block of them).  The launch
// overlaps the end of the kernel before it (a programmatic dependency), which the
// first line waits for.
template <int D, int W>
__global__ void __launch_bounds__(W == 1 ? 256 : W * 32) join_kernel(const Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if constexpr (W > 1) {
    __shared__ float part[W][D];
    __shared__ float2 part_ml[W];
    if (to_join(p, blockIdx.x)) join_row<D, W>(p, blockIdx.x, part, part_ml);
  } else {
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (to_join(p, row)) join_row<D, 1>(p, row, nullptr, nullptr);
  }
}

// Joins tc_kernel's parts (and rows_kernel's chunks of the caches, in a folded
// call): a thread per row of a 128-row tile, F features of it.  FEW tiles are cut
// into many parts, and the time is the latency of their loads in turn: 8 features a
// thread and 8 parts in flight hide it (128 rows over 66,845 keys: 77-80 us with
// tc_kernel, 85 with 32 features and a part at a time; 7 requests of 45 tokens: 41
// and 48).  Many tiles fill the GPU with 32 features, in longer runs of a row (3 x
// 515 tokens: 107 us, 112 with 8; 8 x 300 over 8,191 + 1,030 keys: 191 and 204).
// Rows whose output is written already leave at once.
template <int D, bool FEW>
__global__ void __launch_bounds__(128) join_tiles_kernel(const Params p, const TcPlan tc) {
  constexpr int F = FEW ? 8 : 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int i = threadIdx.x, block = blockIdx.x, f0 = blockIdx.y * F;
  const int rk = block / tc.tiles, req = rk / p.kv_heads, kh = rk - req * p.kv_heads;
  const Row w = tile_row(p, tc, kh, req, block - rk * tc.tiles, i);
  if (!w.live) return;
  const float2* tml = p.tc_ml + (int64_t)block * 128 + i;
  const int64_t tstep = (int64_t)tc.blocks * 128;
  const float2 first = tml[0];
  // part s is the CTA's that begins the item, or of one behind it (inside the grid, whatever a wait that gave up left)
  const int cta0 = max(p.tc_first[block], 0);
  if (first.y == kWritten) return;
  const int64_t row = row_index(p, w);
  const int slots = p.s1 + p.s2;
  float mx = first.x;
#pragma unroll FEW ? 8 : 4
  for (int s = 1; s < tc.slots; ++s) mx = fmaxf(mx, tml[s * tstep].x);
#pragma unroll FEW ? 8 : 4
  for (int s = 0; s < slots; ++s) mx = fmaxf(mx, p.ws_ml[s * p.rows + row].x);
  float l = 0.f, v[F];
#pragma unroll
  for (int u = 0; u < F; ++u) v[u] = 0.f;
  // one part: its weight, and where it wrote any output, that
  auto weight = [&](const float2 ml) {
    const float f = ml.x > -INFINITY ? exp2f(ml.x - mx) : 0.f;
    l = fmaf(ml.y, f, l);
    return f;
  };
  auto add = [&](float f, const float4* x) {
#pragma unroll
    for (int u = 0; u < F / 4; ++u) {
      v[4 * u] = fmaf(f, x[u].x, v[4 * u]);
      v[4 * u + 1] = fmaf(f, x[u].y, v[4 * u + 1]);
      v[4 * u + 2] = fmaf(f, x[u].z, v[4 * u + 2]);
      v[4 * u + 3] = fmaf(f, x[u].w, v[4 * u + 3]);
    }
  };
  auto join = [&](int n, const float2* ml, int64_t ml_step, auto o, auto f_step) {   // o(s): part s's features
    if constexpr (FEW) {
      constexpr int AHEAD = 8;
      for (int s0 = 0; s0 < n; s0 += AHEAD) {
        float f[AHEAD];
        float4 x[AHEAD][F / 4];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) f[a] = weight(s0 + a < n ? ml[(s0 + a) * ml_step] : make_float2(-INFINITY, 0.f));
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
#pragma unroll
          for (int u = 0; u < F / 4; ++u)
            x[a][u] = f[a] > 0.f ? o(s0 + a)[u * f_step] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) add(f[a], x[a]);
      }
    } else {
      constexpr int kUnroll = decltype(f_step)::value == 1 ? 4 : 1;   // a request's chunks are many, a tile's parts two or three
#pragma unroll kUnroll
      for (int s = 0; s < n; ++s) {
        const float f = weight(ml[s * ml_step]);
        if (f > 0.f) {
          float4 x[F / 4];
#pragma unroll
          for (int u = 0; u < F / 4; ++u) x[u] = o(s)[u * f_step];
          add(f, x);
        }
      }
    }
  };
  const int second = tc.halves ? 0 : (block - rk * tc.tiles) & 1;
  const float4* to = p.tc_o + f0 / 4 * 128 + i;
  join(tc.slots, tml, tstep,
       [&](int s) { return to + part_tile(tc, block, second, min(cta0 + s, tc.ctas - 1), s == 0) * (D / 4 * 128); },
       std::integral_constant<int, 128>());
  const float4* wo = reinterpret_cast<const float4*>(p.ws_o + row * D + f0);
  join(slots, p.ws_ml + row, p.rows, [&](int s) { return wo + s * p.rows * (D / 4); }, std::integral_constant<int, 1>());
  const float inv = l == 0.f ? 0.f : 1.f / l;   // no key: zero (a NaN stays one)
  uint4* dst = reinterpret_cast<uint4*>(p.o + w.r * p.o_sr + w.h * p.o_sh + w.m * p.o_sm + f0);
#pragma unroll
  for (int u = 0; u < F / 8; ++u)
    dst[u] = make_uint4(pack_bf16x2(v[8 * u] * inv, v[8 * u + 1] * inv), pack_bf16x2(v[8 * u + 2] * inv, v[8 * u + 3] * inv),
                        pack_bf16x2(v[8 * u + 4] * inv, v[8 * u + 5] * inv), pack_bf16x2(v[8 * u + 6] * inv, v[8 * u + 7] * inv));
  if (p.lse && f0 == 0) p.lse[w.r * p.lse_sr + w.h * p.lse_sh + w.m] = l == 0.f ? -INFINITY : mx + log2f(l);
}

// A launch that may begin before the kernel ahead of it in the stream has ended.
template <typename... P, typename... A>
static int launch_early(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, const A&... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return fail(GPA_ERR_CUDA, "gpa_attention_shared_prefix: %s", cudaGetErrorString(e));
  return check_launch("gpa_attention_shared_prefix");
}

// How a call is cut into items.
struct Plan {
  bool rows_run, tc_run;
  int wm1, rt1, s1, wm2, rt2, s2, chunk;
  int64_t items, rows;
  TcPlan tc;
  int64_t bytes(int head_dim) const {   // of the partial outputs, in whole ones of a row
    const int64_t tiles = tc_run ? part_tiles(tc) * 128 * head_dim + (int64_t)tc.blocks * (tc.slots * 256 + 1) : 0;
    return ((tiles + head_dim + 1) / (head_dim + 2) + (s1 + s2) * rows) * (head_dim + 2) * 4;
  }
};

static int warps_for(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

// The tensor-core kernel's share: over prefix and own keys of each request, or
// folded over the prefix alone.  False where its counts would not fit, or a token's
// query heads of one key head a 128-row tile.
static bool plan_tc(TcPlan* tc, bool fold, int requests, int queries, int group, int kv_heads, int64_t prefix_tiles,
                    int64_t cache_tiles, int64_t* total) {
  if (group > 128) return false;
  const int64_t tokens = fold ? (int64_t)requests * queries : queries;
  tc->fold = fold;
  tc->tokens = (int)tokens;
  tc->per_tile = 128 / group;
  const int64_t tiles = (tokens + tc->per_tile - 1) / tc->per_tile;
  const int64_t heads = (int64_t)kv_heads * (fold ? 1 : requests);
  tc->tiles = (int)tiles;
  tc->halves = tiles == 1;
  // The units of all items at full lengths (the kernel counts the real ones), and
  // what a CTA gets of them.  An item is cut where a span ends, into at most
  // units / span + 2 parts; twice the units / span leaves room for spans that
  // shorter lengths make shorter.
  const int64_t keys = std::max<int64_t>(prefix_tiles + (fold ? 0 : cache_tiles), 1);
  const int64_t steps = tc->halves ? (keys + 1) / 2 : keys;
  const int each = tiles > 1 ? kPair : kSingle;
  const int64_t units = (steps + kItemSteps) * each, least = std::min<int64_t>(kLeastSteps, steps) * each;
  if ((double)(tiles + 1) * kPair * (steps + kItemSteps) * heads >= 1e9 || (double)tiles * heads >= 1e7) return false;
  *total = (tiles / 2 * kPair + tiles % 2 * kSingle) * (steps + kItemSteps) * heads;
  const int64_t span = std::max((*total + kSms - 1) / kSms, least);
  const int64_t cuts = std::min(2 * ((units + span - 1) / span), std::max<int64_t>(units / least, 1));
  tc->blocks = (int)(tiles * heads);
  tc->least = (int)std::max((units + cuts - 1) / cuts, least);
  tc->ctas = (int)std::min<int64_t>(kSms, (*total + least - 1) / least);
  tc->slots = (int)((units + tc->least - 1) / tc->least) + 1;
  return true;
}

// joint, fold: whether the tensor-core kernel can take the call in that form.
static Plan make_plan(int requests, int queries, int heads, int kv_heads, int head_dim, int prefix, int cache,
                      bool joint, bool fold) {
  Plan p{};
  const int group = heads / kv_heads;
  const int64_t r1 = (int64_t)requests * queries * group, r2 = (int64_t)queries * group;
  const int64_t t1 = (prefix + BN - 1) / BN, t2 = (cache + BN - 1) / BN;
  p.rows = r1 * kv_heads;
  // Which kernels: the least time by a model in units of half a microsecond of an
  // SM at head_dim 64 (twice that at 128).  A 64-key tile of rows_kernel takes 0.9,
  // 1.2 or 1.6 for 16, 32 or 64 rows; caches on fewer rows than the prefix wait for
  // HBM while its products run, and cost a third less beside it (64 requests over
  // 66,845 + 1,374 keys: 127 us, where each alone takes 95 and 64).  A step of
  // tc_kernel takes 3 or 2.4, in halves 4.5, and starting and ending take 20 on every
  // SM, another launch for the caches 10.  Measured on both sides (16 heads, 66,845
  // keys, us): 32 rows 62 here; 48 rows 93 and 76 there, 64 rows 95 and 76, 128 rows
  // 166 and 77; 64 rows with caches of 300 100 and 95, of 1,374 127 and 144.
  auto rows_cost = [&](int64_t rows, int64_t tiles) {
    const int wm = warps_for(rows);
    return (double)((rows + 16 * wm - 1) / (16 * wm)) * tiles * (wm == 1 ? 0.9 : wm == 2 ? 1.2 : 1.6) * kv_heads;
  };
  const double own_cost = requests * rows_cost(r2, t2);
  double least = rows_cost(r1, t1) + own_cost * (prefix > 0 && warps_for(r2) < warps_for(r1) ? 0.65 : 1.0);
  TcPlan tc{};
  int64_t total = 0;
  const int64_t k1 = (prefix + 127) / 128, k2 = (cache + 127) / 128;
  for (int way = 0; way < 2; ++way) {   // joint, folded
    if (!(way ? fold && prefix > 0 : joint && prefix + (int64_t)cache > 0)) continue;
    if (!plan_tc(&tc, way, requests, queries, group, kv_heads, k1, k2, &total)) continue;
    const double cost = total * (tc.halves ? 4.5 / kSingle : 3.0 / kPair) + 20.0 * kSms +
                        (way && cache > 0 ? own_cost + 10.0 * kSms : 0.0);
    if (cost < least) {
      least = cost;
      p.tc = tc;
      p.tc_run = true;
    }
  }
  p.rows_run = !p.tc_run || (p.tc.fold && cache > 0);
  if (p.rows_run) {
    const int64_t tiles1 = p.tc_run ? 0 : t1;
    p.wm1 = p.tc_run ? 4 : warps_for(r1);
    p.wm2 = warps_for(r2);
    p.rt1 = p.tc_run ? 0 : (int)((r1 + p.wm1 * 16 - 1) / (p.wm1 * 16));
    p.rt2 = (int)((r2 + p.wm2 * 16 - 1) / (p.wm2 * 16));
    const int64_t units = kv_heads * (p.rt1 * tiles1 + (int64_t)requests * p.rt2 * t2);
    // two items per resident CTA: short enough to even out requests of unequal
    // lengths, long enough that the partial outputs are a small share
    const int64_t want = (int64_t)kSms * resident(head_dim, p.wm1, p.wm2) * 2;
    const int64_t per = std::max<int64_t>((units + want - 1) / want, kSlotTiles);
    p.chunk = (int)std::min<int64_t>(per, 1 << 24) * BN;
    p.s1 = (int)((tiles1 + per - 1) / per);
    p.s2 = (int)((t2 + per - 1) / per);
    p.items = kv_heads * ((int64_t)p.rt1 * p.s1 + (int64_t)requests * p.rt2 * p.s2);
  }
  p.tc.keep = p.tc_run && p.s2 > 0;
  return p;
}

template <int D, int WM1, int WM2>
static int launch_rows(const Params& p, int64_t items, bool early, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(rows_kernel<D, WM1, WM2>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::SMEM);
  if (e != cudaSuccess) return fail(GPA_ERR_CUDA, "gpa_attention_shared_prefix: %s", cudaGetErrorString(e));
  if (early) return launch_early(rows_kernel<D, WM1, WM2>, dim3((unsigned)items), THREADS, Cfg<D>::SMEM, st, p);
  rows_kernel<D, WM1, WM2><<<(unsigned)items, THREADS, Cfg<D>::SMEM, st>>>(p);
  return check_launch("gpa_attention_shared_prefix");
}

template <int D>
static int launch(const Params& p, const Plan& plan, cudaStream_t st) {
  int rc = GPA_OK;
  const bool tc = plan.tc_run;
  if (tc) rc = launch_tc(p, D, plan.tc, st);
  if (!rc && plan.rows_run && plan.items > 0) {
    switch (plan.wm1 * 8 + plan.wm2) {   // wm2 <= wm1: own rows are part of the prefix's
      case 1 * 8 + 1: rc = launch_rows<D, 1, 1>(p, plan.items, tc, st); break;
      case 2 * 8 + 1: rc = launch_rows<D, 2, 1>(p, plan.items, tc, st); break;
      case 2 * 8 + 2: rc = launch_rows<D, 2, 2>(p, plan.items, tc, st); break;
      case 4 * 8 + 1: rc = launch_rows<D, 4, 1>(p, plan.items, tc, st); break;
      case 4 * 8 + 2: rc = launch_rows<D, 4, 2>(p, plan.items, tc, st); break;
      default: rc = launch_rows<D, 4, 4>(p, plan.items, tc, st); break;
    }
  }
  if (rc) return rc;
  if (tc && (int64_t)plan.tc.blocks * (D / 8) <= kJoinCtas)
    return launch_early(join_tiles_kernel<D, true>, dim3(plan.tc.blocks, D / 8), 128, 0, st, p, plan.tc);
  if (tc) return launch_early(join_tiles_kernel<D, false>, dim3(plan.tc.blocks, D / 32), 128, 0, st, p, plan.tc);
  const int slots = p.s1 + p.s2;
  auto join = [&](auto w) {
    constexpr int W = decltype(w)::value;
    return launch_early(join_kernel<D, W>, dim3((unsigned)p.rows), W * 32, 0, st, p);
  };
  // Warps per row: as many as its chunks feed, while the rows alone do not fill the
  // GPU.  With the kernel before, us, at 32, 8, 4, 2 and 1 warps: one head over
  // 200,000 keys (592 chunks) 25, 33; 16 rows of 16 heads over 66,845 (75) -, 55, 56,
  // 59; 12 rows of 16 heads over 4,000 (11) -, 15.7, 14.0, 14.6, 20; 18 x 2 tokens of
  // 64 heads (10) -, 22, 18.7, 16.5, 17.4; 8 x 64 tokens of 16 -, 56, 43, 36, 32.
  if (slots > 128) return join(std::integral_constant<int, 32>());
  if (slots > 32) return join(std::integral_constant<int, 8>());
  if (slots > 4 && p.rows <= 1280) return join(std::integral_constant<int, 4>());
  if (slots > 4 && p.rows <= 3000) return join(std::integral_constant<int, 2>());
  return launch_early(join_kernel<D, 1>, dim3((unsigned)((p.rows + 7) / 8)), 256, 0, st, p);
}

static int check_sizes(const char* what, int requests, int queries, int heads, int kv_heads, int head_dim, int prefix,
                       int cache) {
  if (requests < 0 || queries < 0 || heads <= 0 || kv_heads <= 0 || prefix < 0 || cache < 0 || heads % kv_heads)
    return fail(GPA_ERR_INVALID, "%s: bad sizes (heads must be a multiple of kv_heads)", what);
  if (head_dim != 64 && head_dim != 128) return fail(GPA_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128", what);
  if ((double)requests * queries * heads >= 2147483648.0)
    return fail(GPA_ERR_UNSUPPORTED, "%s: 2^31 or more query rows", what);
  if (prefix > (1 << 30) || cache > (1 << 30)) return fail(GPA_ERR_UNSUPPORTED, "%s: more than 2^30 keys", what);
  return GPA_OK;
}

}  // namespace prefix
}  // namespace gpa

using namespace gpa;

extern "C" int64_t gpa_attention_shared_prefix_workspace_bytes(int requests, int queries, int heads, int kv_heads,
                                                               int head_dim, int prefix, int cache) {
  if (prefix::check_sizes("gpa_attention_shared_prefix_workspace_bytes", requests, queries, heads, kv_heads, head_dim,
                          prefix, cache))
    return -1;
  if (requests == 0 || queries == 0) return 0;
  // strides decide which kernels can run: room for each way
  int64_t bytes = 0;
  for (int way = 0; way < 4; ++way)
    bytes = std::max(bytes, prefix::make_plan(requests, queries, heads, kv_heads, head_dim, prefix, cache, way & 1,
                                              way & 2).bytes(head_dim));
  return bytes;
}

extern "C" int64_t gpa_attention_shared_prefix_call_bytes(
    int64_t q_sr, int64_t q_sh, int64_t q_sm, int64_t kp_sh, int64_t kp_sn, int64_t vp_sh, int64_t vp_sn, int64_t ko_sr,
    int64_t ko_sh, int64_t ko_sn, int64_t vo_sr, int64_t vo_sh, int64_t vo_sn, int requests, int queries, int heads,
    int kv_heads, int head_dim, int prefix_len, int cache_len, float sm_scale) {
  if (prefix::check_sizes("gpa_attention_shared_prefix_call_bytes", requests, queries, heads, kv_heads, head_dim,
                          prefix_len, cache_len))
    return -1;
  if (requests == 0 || queries == 0) return 0;
  prefix::Params p{};
  p.requests = requests; p.queries = queries; p.heads = heads; p.kv_heads = kv_heads; p.group = heads / kv_heads;
  p.prefix = prefix_len; p.cache = cache_len;
  p.q_sr = q_sr; p.q_sh = q_sh; p.q_sm = q_sm;
  p.kp_sh = kp_sh; p.kp_sn = kp_sn; p.vp_sh = vp_sh; p.vp_sn = vp_sn;
  p.ko_sr = ko_sr; p.ko_sh = ko_sh; p.ko_sn = ko_sn;
  p.vo_sr = vo_sr; p.vo_sh = vo_sh; p.vo_sn = vo_sn;
  p.scale = sm_scale;
  return prefix::make_plan(requests, queries, heads, kv_heads, head_dim, prefix_len, cache_len,
                           prefix::tc_takes(p, head_dim, false), prefix::tc_takes(p, head_dim, true)).bytes(head_dim);
}

extern "C" int gpa_attention_shared_prefix(
    const void* q, int64_t q_sr, int64_t q_sh, int64_t q_sm, const void* k_prefix, int64_t kp_sh, int64_t kp_sn,
    const void* v_prefix, int64_t vp_sh, int64_t vp_sn, const float* bias, int64_t bias_sh, const void* k_own,
    int64_t ko_sr, int64_t ko_sh, int64_t ko_sn, const void* v_own, int64_t vo_sr, int64_t vo_sh, int64_t vo_sn,
    const int32_t* own_len, const int32_t* q_len, int requests, int queries, int heads, int kv_heads, int head_dim,
    int prefix_len, int cache_len, float sm_scale, int causal, void* o, int64_t o_sr, int64_t o_sh, int64_t o_sm,
    float* lse, int64_t lse_sr, int64_t lse_sh, void* workspace, int64_t workspace_bytes, int* status, void* stream) {
  const char* what = "gpa_attention_shared_prefix";
  int rc = prefix::check_sizes(what, requests, queries, heads, kv_heads, head_dim, prefix_len, cache_len);
  if (rc) return rc;
  if (requests == 0 || queries == 0) return ok();
  if (!q || !o || (prefix_len && (!k_prefix || !v_prefix)) || (cache_len && (!k_own || !v_own)))
    return fail(GPA_ERR_INVALID, "%s: null pointer", what);
  if (!aligned16(q) || !aligned16(o) || !aligned16(k_prefix) || !aligned16(v_prefix) || !aligned16(k_own) ||
      !aligned16(v_own))
    return fail(GPA_ERR_INVALID, "%s: q, keys, values and o must be 16-byte aligned", what);
  if ((q_sr | q_sh | q_sm | kp_sh | kp_sn | vp_sh | vp_sn | ko_sr | ko_sh | ko_sn | vo_sr | vo_sh | vo_sn | o_sr |
       o_sh | o_sm) & 7)
    return fail(GPA_ERR_INVALID, "%s: strides must be multiples of 8", what);
  if (!prefix_len) bias = nullptr;
  prefix::Params p;
  p.q = (const __nv_bfloat16*)q;
  p.kp = (const __nv_bfloat16*)k_prefix;
  p.vp = (const __nv_bfloat16*)v_prefix;
  p.ko = (const __nv_bfloat16*)k_own;
  p.vo = (const __nv_bfloat16*)v_own;
  p.bias = bias;
  p.own_len = own_len;
  p.q_len = q_len;
  p.requests = requests;
  p.queries = queries;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.group = heads / kv_heads;
  p.prefix = prefix_len;
  p.cache = cache_len;
  p.q_sr = q_sr; p.q_sh = q_sh; p.q_sm = q_sm;
  p.kp_sh = kp_sh; p.kp_sn = kp_sn; p.vp_sh = vp_sh; p.vp_sn = vp_sn;
  p.ko_sr = ko_sr; p.ko_sh = ko_sh; p.ko_sn = ko_sn;
  p.vo_sr = vo_sr; p.vo_sh = vo_sh; p.vo_sn = vo_sn;
  p.bias_sh = bias_sh;
  p.scale = sm_scale;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.causal = causal;
  p.o = (__nv_bfloat16*)o;
  p.o_sr = o_sr; p.o_sh = o_sh; p.o_sm = o_sm;
  p.lse = lse;
  p.lse_sr = lse_sr; p.lse_sh = lse_sh;
  const prefix::Plan plan =
      prefix::make_plan(requests, queries, heads, kv_heads, head_dim, prefix_len, cache_len,
                        prefix::tc_takes(p, head_dim, false), prefix::tc_takes(p, head_dim, true));
  if (plan.items >= (1ll << 31))
    return fail(GPA_ERR_UNSUPPORTED, "%s: too many work items", what);
  const int64_t bytes = plan.bytes(head_dim);
  if (bytes && (!workspace || !aligned16(workspace) || workspace_bytes < bytes))
    return fail(GPA_ERR_INVALID, "%s: workspace missing, unaligned or too small", what);
  p.status = status;
  p.rt1 = plan.rt1; p.s1 = plan.s1; p.rt2 = plan.rt2; p.s2 = plan.s2; p.chunk = plan.chunk;
  p.rows = plan.rows;
  // the tiles' outputs (whole lines each), the rows', their maxima and sums, then the items' first CTAs
  p.tc_o = (float4*)workspace;
  p.ws_o = (float*)workspace + (plan.tc_run ? prefix::part_tiles(plan.tc) * 128 * head_dim : 0);
  p.tc_ml = reinterpret_cast<float2*>(p.ws_o + (plan.s1 + plan.s2) * plan.rows * head_dim);
  p.ws_ml = p.tc_ml + (plan.tc_run ? (int64_t)plan.tc.slots * plan.tc.blocks * 128 : 0);
  p.tc_first = reinterpret_cast<int32_t*>(p.ws_ml + (plan.s1 + plan.s2) * plan.rows);
  cudaStream_t st = (cudaStream_t)stream;
  return head_dim == 64 ? prefix::launch<64>(p, plan, st) : prefix::launch<128>(p, plan, st);
}
