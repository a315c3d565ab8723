// The residual stream between two sub-blocks, in one pass:
//   z = x + gate * P(y)     P: identity, LayerNorm or RMSNorm of the branch output y
//   h = N(z)                N: LayerNorm or RMSNorm in front of the next sub-block
// and its gradients.  With d = dz + N'(dh):
//   dx = d, dgate = sum d * P(y), dy = P'(gate * d), norm weights and biases:
//   column sums over the rows.
//
// Both directions are bound by HBM: forward reads x, y and writes z, h; backward
// reads dz, dh, z, y and writes dx, dy.  Everything of a row stays in registers
// between its load and its store, and all arithmetic is fp32.
//
// Roundings: z is kept in the stream's type and N normalises z as kept; without
// a norm of the branch, gate * y is rounded to the stream's type before the add.
// For a bf16 stream these are the roundings of residual_scale followed by
// layernorm (norm.cu), so a block that changes from the two kernels to this one
// keeps its results bit for bit (at layernorm's widths up to 2,048 columns, where
// the sums also run in the same order).
#include "common.cuh"
#include "capi_util.h"

namespace gpa {
namespace resnorm {

enum : int { kNone = GPA_NORM_NONE, kLayer = GPA_NORM_LAYER, kRms = GPA_NORM_RMS };

// 8 consecutive elements as they lie in memory, and as floats.
template <typename T>
struct Raw8;
template <>
struct Raw8<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { a = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void get(float* v) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float* v) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
};

__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* v) {
  uint4 r;
  r.x = pack_bf16x2(v[0], v[1]);
  r.y = pack_bf16x2(v[2], v[3]);
  r.z = pack_bf16x2(v[4], v[5]);
  r.w = pack_bf16x2(v[6], v[7]);
  *reinterpret_cast<uint4*>(p) = r;
}
__device__ __forceinline__ void store8(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *(reinterpret_cast<float4*>(p) + 1) = make_float4(v[4], v[5], v[6], v[7]);
}

// Gate and norm parameters come in fp32 or bf16, told apart at run time (the
// branch is uniform and the rows stay in cache).
struct Param {
  const void* p;
  int bf16;
  __device__ __forceinline__ explicit operator bool() const { return p != nullptr; }
  __device__ __forceinline__ void get(int64_t i, float* v) const {
    if (bf16) {
      Raw8<__nv_bfloat16> r;
      r.a = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p) + i));
      r.get(v);
    } else {
      const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
      const float4 a = __ldg(q), b = __ldg(q + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
  }
};

template <typename T>
__device__ __forceinline__ float round_to(float v) { return v; }
template <>
__device__ __forceinline__ float round_to<__nv_bfloat16>(float v) {
  return __bfloat162float(__float2bfloat16_rn(v));
}

struct FwdParams {
  const void *x, *y;
  void *z, *h;
  int64_t xs, ys, zs, hs;
  Param gate;
  int64_t gate_rows;   // rows that share one gate row
  int rows, cols;
  int post_kind, kind;
  Param pw, pb, w, b;
  float post_eps, eps;
  float* stats;        // [rows, 4]: mean, 1/std of y; mean, 1/std of z (or null)
};

// Sums over the WPR warps that share a row, two at a time.  Every warp of the
// row's group calls it the same number of times; two buffers in turn make one
// barrier enough.
template <int WPR>
struct RowSum {
  float2* buf;   // [2][WPR] of this group
  int bar, turn;
  __device__ __forceinline__ float2 operator()(float a, float b) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if constexpr (WPR > 1) {
      float2* w = buf + turn * WPR;
      turn ^= 1;
      const int warp = (threadIdx.x >> 5) % WPR;
      if ((threadIdx.x & 31) == 0) w[warp] = make_float2(a, b);
      asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(WPR * 32) : "memory");
      a = b = 0.f;
#pragma unroll
      for (int i = 0; i < WPR; ++i) {
        a += w[i].x;
        b += w[i].y;
      }
    }
    return make_float2(a, b);
  }
  __device__ __forceinline__ float operator()(float a) { return (*this)(a, 0.f).x; }
};

// Forward.  WPR warps per row, VPL vectors of 8 columns per lane; a lane's
// vectors past the row's end stay zero and are never loaded or stored.  A bf16
// stream without a norm of the branch takes one warp per row up to 2,048 columns:
// the sums are shuffles in layernorm's order, and 274,800 x 1,024 takes 372 us
// (94% of the measured copy rate).  Elsewhere a lane takes at most four vectors,
// two of fp32: 110,000 x 1,024 with an fp32 stream and a normed bf16 branch takes
// 249 us (251 with two, 311 with one), with an fp32 branch 300 (365 with four).
template <int VPL, int WPR, typename TX, typename TY>
__global__ void __launch_bounds__(256) fwd_kernel(const FwdParams p) {
  __shared__ float2 red[8 / WPR][2 * WPR];
  const int t = threadIdx.x % (WPR * 32), grp = threadIdx.x / (WPR * 32);
  const int64_t row = (int64_t)blockIdx.x * (8 / WPR) + grp;
  if (row >= p.rows) return;   // whole groups leave together
  RowSum<WPR> sum{red[grp], 1 + grp, 0};
  const TX* xr = reinterpret_cast<const TX*>(p.x) + row * p.xs;
  const TY* yr = reinterpret_cast<const TY*>(p.y) + row * p.ys;
  const float n = (float)p.cols;
  Raw8<TX> xv[VPL];
  Raw8<TY> yv[VPL];
  bool in[VPL];
#pragma unroll
  for (int u = 0; u < VPL; ++u) {
    const int c = (u * WPR * 32 + t) * 8;
    in[u] = c < p.cols;
    if (in[u]) {
      xv[u].load(xr + c);
      yv[u].load(yr + c);
    } else {
      xv[u].zero();
      yv[u].zero();
    }
  }
  float mean_y = 0.f, rstd_y = 1.f;
  if (p.post_kind != kNone) {
    if (p.post_kind == kLayer) {
      float s = 0.f;
#pragma unroll
      for (int u = 0; u < VPL; ++u) {
        float v[8];
        yv[u].get(v);
#pragma unroll
        for (int i = 0; i < 8; i += 2) s += v[i] + v[i + 1];
      }
      mean_y = sum(s) / n;
    }
    float q = 0.f;
#pragma unroll
    for (int u = 0; u < VPL; ++u) {
      float v[8];
      yv[u].get(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = in[u] ? v[i] - mean_y : 0.f;
        q = fmaf(d, d, q);
      }
    }
    rstd_y = rsqrtf(sum(q) / n + p.post_eps);
  }
  const int64_t grow = p.gate ? (int64_t)((uint32_t)row / (uint32_t)p.gate_rows) * p.cols : 0;
  float z[VPL][8];
  float s = 0.f;
  TX* zr = reinterpret_cast<TX*>(p.z) + row * p.zs;
#pragma unroll
  for (int u = 0; u < VPL; ++u) {
    const int c = (u * WPR * 32 + t) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) z[u][i] = 0.f;
    if (in[u]) {
      float v[8], w8[8];
      yv[u].get(v);
      if (p.post_kind != kNone) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (v[i] - mean_y) * rstd_y;
        if (p.pw) {
          p.pw.get(c, w8);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] *= w8[i];
        }
        if (p.pb) {
          p.pb.get(c, w8);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += w8[i];
        }
      }
      if (p.gate) {
        p.gate.get(grow + c, w8);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], w8[i]);
      }
      float x8[8];
      xv[u].get(x8);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        z[u][i] = round_to<TX>(__fadd_rn(x8[i], p.post_kind == kNone ? round_to<TX>(v[i]) : v[i]));
      store8(zr + c, z[u]);
    }
#pragma unroll
    for (int i = 0; i < 8; i += 2) s += z[u][i] + z[u][i + 1];
  }
  float mean = 0.f, rstd = 1.f;
  if (p.kind != kNone) {
    if (p.kind == kLayer) mean = sum(s) / n;
    float q = 0.f;
#pragma unroll
    for (int u = 0; u < VPL; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = in[u] ? z[u][i] - mean : 0.f;
        q = fmaf(d, d, q);
      }
    rstd = rsqrtf(sum(q) / n + p.eps);
    TY* hr = reinterpret_cast<TY*>(p.h) + row * p.hs;
#pragma unroll
    for (int u = 0; u < VPL; ++u) {
      const int c = (u * WPR * 32 + t) * 8;
      if (!in[u]) continue;
      float w8[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f}, b8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (p.w) p.w.get(c, w8);
      if (p.b) p.b.get(c, b8);
#pragma unroll
      for (int i = 0; i < 8; ++i) w8[i] = fmaf((z[u][i] - mean) * rstd, w8[i], b8[i]);
      store8(hr + c, w8);
    }
  }
  if (p.stats && t == 0)
    *reinterpret_cast<float4*>(p.stats + row * 4) = make_float4(mean_y, rstd_y, mean, rstd);
}

// Column-sum slots of the backward pass.
enum : int { kGate = 0, kW = 1, kB = 2, kPw = 3, kPb = 4, kSlots = 5 };

struct BwdParams {
  const void *dz, *dh, *z, *y;   // dz or dh may be null (a zero gradient)
  void *dx, *dy;
  int64_t dzs, dhs, zs, ys, dxs, dys;
  Param gate;
  int64_t gate_rows;
  int rows, cols;
  int post_kind, kind;
  Param pw, pb, w;
  const float* stats;
  int want[kSlots];    // which column sums the caller takes
  int whole;           // each worker takes whole gate groups and writes their gate gradient itself
  int groups, per_group, workers;   // split: per_group workers in each of `groups` gate groups
  void* dgate;         // whole groups: [groups, cols]
  int dgate_bf16;
  float* part;         // [workers][kSlots][cols]
};

// Backward.  A group of WPR warps is one worker: it walks rows, each thread
// owning the same VPT x 8 columns of all of them, so the column sums stay in its
// registers until the end (one partial per worker, added up by sum_kernel in a
// fixed order: no atomics, the same bits every time).  The next row's vectors
// are loaded before this row's sums are exchanged.
template <bool POST, int WPR, int VPT, typename TX, typename TY>
__global__ void __launch_bounds__(WPR * 32 < 128 ? 128 : WPR * 32) bwd_kernel(const BwdParams p) {
  constexpr int NG = WPR * 32 < 128 ? 128 / (WPR * 32) : 1;
  asm volatile("griddepcontrol.launch_dependents;");   // the column sums may be launched, and wait for this grid's end
  __shared__ float2 red[NG][2 * WPR];
  const int grp = threadIdx.x / (WPR * 32);
  const int t = threadIdx.x % (WPR * 32);
  const int worker = blockIdx.x * NG + grp;
  if (worker >= p.workers) return;
  RowSum<WPR> sum{red[grp], 1 + grp, 0};
  // rows of this worker: first, step, end (split), or whole gate groups in turn
  int64_t row, step, end;
  int g = 0;
  if (p.whole) {
    g = worker;
    row = (int64_t)g * p.gate_rows;
    step = 1;
    end = row + p.gate_rows;
  } else {
    g = worker / p.per_group;
    row = (int64_t)g * p.gate_rows + worker % p.per_group;
    step = p.per_group;
    end = (int64_t)(g + 1) * p.gate_rows;
  }
  const float inv_n = 1.f / (float)p.cols;
  float acc[POST ? kSlots : 3][VPT][8];
#pragma unroll
  for (int k = 0; k < (POST ? kSlots : 3); ++k)
#pragma unroll
    for (int u = 0; u < VPT; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[k][u][i] = 0.f;

  Raw8<TX> dzr[VPT], zr[VPT];
  Raw8<TY> dhr[VPT], yr[VPT];
  float4 st;
  auto load_row = [&](int64_t r) {
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      const int c = (u * WPR * 32 + t) * 8;
      const bool in = c < p.cols;
      if (in && p.dz) dzr[u].load(reinterpret_cast<const TX*>(p.dz) + r * p.dzs + c); else dzr[u].zero();
      if (in && p.dh) {
        dhr[u].load(reinterpret_cast<const TY*>(p.dh) + r * p.dhs + c);
        zr[u].load(reinterpret_cast<const TX*>(p.z) + r * p.zs + c);
      } else {
        dhr[u].zero();
        zr[u].zero();
      }
      if (in) yr[u].load(reinterpret_cast<const TY*>(p.y) + r * p.ys + c); else yr[u].zero();
    }
    st = __ldg(reinterpret_cast<const float4*>(p.stats) + r);
  };
  if (row < end) load_row(row);
  while (row < end) {
    const float mean_y = st.x, rstd_y = st.y;
    const float mean = p.dh ? st.z : 0.f, rstd = p.dh ? st.w : 0.f;   // h unused: nothing comes through its norm, not even NaN
    float d[VPT][8], y8[VPT][8];
    float s1 = 0.f, s2 = 0.f;
    // N': the gradient through the norm of z
    float gw[VPT][8], zh[VPT][8];
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      const int c = (u * WPR * 32 + t) * 8;
      float w8[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f}, dh8[8];
      if (p.w && c < p.cols) p.w.get(c, w8);
      dhr[u].get(dh8);
      zr[u].get(zh[u]);
      dzr[u].get(d[u]);
      yr[u].get(y8[u]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        zh[u][i] = (zh[u][i] - mean) * rstd;
        acc[kW][u][i] = fmaf(dh8[i], zh[u][i], acc[kW][u][i]);
        acc[kB][u][i] += dh8[i];
        gw[u][i] = dh8[i] * w8[i];
        s1 += gw[u][i];
        s2 = fmaf(gw[u][i], zh[u][i], s2);
      }
    }
    const int64_t cur = row;
    row += step;
    int64_t next = row;
    int next_g = g;
    if (p.whole && next >= end) {   // the next whole group of this worker
      next_g = g + p.workers;
      next = (int64_t)next_g * p.gate_rows;
    }
    const bool more = p.whole ? next_g < p.groups : next < end;
    if (more) load_row(next);
    if (p.dh) {
      const float2 s = sum(s1, s2);
      s1 = p.kind == kLayer ? s.x * inv_n : 0.f;
      s2 = s.y * inv_n;
    }
    float t1 = 0.f, t2 = 0.f;
    const int64_t grow = p.gate ? (int64_t)g * p.cols : 0;
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      const int c = (u * WPR * 32 + t) * 8;
      const bool in = c < p.cols;
#pragma unroll
      for (int i = 0; i < 8; ++i) d[u][i] = fmaf(rstd, gw[u][i] - s1 - zh[u][i] * s2, d[u][i]);
      if (in) store8(reinterpret_cast<TX*>(p.dx) + cur * p.dxs + c, d[u]);
      float g8[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
      if (p.gate && in) p.gate.get(grow + c, g8);
      if constexpr (POST) {
        float pw8[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f}, pb8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (p.pw && in) p.pw.get(c, pw8);
        if (p.pb && in) p.pb.get(c, pb8);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float dd = in ? d[u][i] : 0.f;
          const float yh = (y8[u][i] - mean_y) * rstd_y;
          acc[kGate][u][i] = fmaf(dd, fmaf(yh, pw8[i], pb8[i]), acc[kGate][u][i]);
          const float dp = dd * g8[i];
          acc[kPw][u][i] = fmaf(dp, yh, acc[kPw][u][i]);
          acc[kPb][u][i] += dp;
          y8[u][i] = yh;
          d[u][i] = dp * pw8[i];
          t1 += d[u][i];
          t2 = fmaf(d[u][i], yh, t2);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc[kGate][u][i] = fmaf(d[u][i], y8[u][i], acc[kGate][u][i]);
          d[u][i] *= g8[i];
        }
        if (in) store8(reinterpret_cast<TY*>(p.dy) + cur * p.dys + c, d[u]);
      }
    }
    if constexpr (POST) {
      const float2 s = sum(t1, t2);
      t1 = p.post_kind == kLayer ? s.x * inv_n : 0.f;
      t2 = s.y * inv_n;
#pragma unroll
      for (int u = 0; u < VPT; ++u) {
        const int c = (u * WPR * 32 + t) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) d[u][i] = rstd_y * (d[u][i] - t1 - y8[u][i] * t2);
        if (c < p.cols) store8(reinterpret_cast<TY*>(p.dy) + cur * p.dys + c, d[u]);
      }
    }
    if (p.whole && next_g != g) {   // a gate group is complete
#pragma unroll
      for (int u = 0; u < VPT; ++u) {
        const int c = (u * WPR * 32 + t) * 8;
        if (p.want[kGate] && c < p.cols) {
          if (p.dgate_bf16)
            store8(reinterpret_cast<__nv_bfloat16*>(p.dgate) + (int64_t)g * p.cols + c, acc[kGate][u]);
          else
            store8(reinterpret_cast<float*>(p.dgate) + (int64_t)g * p.cols + c, acc[kGate][u]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[kGate][u][i] = 0.f;
      }
      g = next_g;
      row = next;
      end = more ? row + p.gate_rows : row;
    }
  }
#pragma unroll
  for (int k = 0; k < (POST ? kSlots : 3); ++k) {
    if (!p.want[k] || (k == kGate && p.whole)) continue;
    float* o = p.part + ((int64_t)worker * kSlots + k) * p.cols;
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      const int c = (u * WPR * 32 + t) * 8;
      if (c < p.cols) store8(o + c, acc[k][u]);
    }
  }
}

struct SumParams {
  const float* part;
  int cols, workers, per_group;
  int gate_groups;            // gate rows summed here (split groups), else 0
  void* out[kSlots];
  int bf16[kSlots];
};

// Column sums of the workers' partials: 32 columns x 32 workers per step.
// blockIdx.y: 0-3 the norm parameters, 4.. the gate groups.
__global__ void __launch_bounds__(1024) sum_kernel(const SumParams p) {
  __shared__ float red[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");   // launched before the backward kernel's end
  const int cx = threadIdx.x & 31, wy = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cx;
  const int slot = blockIdx.y < 4 ? (int)blockIdx.y + 1 : kGate;
  const int group = (int)blockIdx.y - 4;
  if (!p.out[slot]) return;
  const int w0 = slot == kGate ? group * p.per_group : 0;
  const int w1 = slot == kGate ? w0 + p.per_group : p.workers;
  float s = 0.f;
  if (c < p.cols) {
    const float* q = p.part + (int64_t)slot * p.cols + c;
#pragma unroll 8
    for (int w = w0 + wy; w < w1; w += 32) s += q[(int64_t)w * kSlots * p.cols];
  }
  red[wy][cx] = s;
  __syncthreads();
  if (wy == 0 && c < p.cols) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += red[i][cx];
    const int64_t at = (slot == kGate ? (int64_t)group * p.cols : 0) + c;
    if (p.bf16[slot])
      reinterpret_cast<__nv_bfloat16*>(p.out[slot])[at] = __float2bfloat16_rn(s);
    else
      reinterpret_cast<float*>(p.out[slot])[at] = s;
  }
}

// How the rows are split among the workers of a backward pass.
struct Split {
  int wpr, vpt, whole, per_group, workers;
};

static Split split_rows(int64_t rows, int cols, int64_t gate_rows) {
  Split s;
  s.vpt = cols > 4096 ? 2 : 1;
  s.wpr = 1;
  while (s.wpr * s.vpt * 256 < cols) s.wpr *= 2;
  const int64_t groups = rows / gate_rows;
  // 16 warps per SM.  (With a branch norm up to 512 columns, and fp32/fp32 up to 1,024,
  // the kernel's 143-165 registers let 12 be resident: the last workers run behind.)
  const int64_t most = std::max<int64_t>(148ll * 16 / s.wpr, 1);
  s.whole = groups >= most;
  if (s.whole) {
    s.per_group = 1;
    s.workers = (int)std::min<int64_t>(groups, most);
  } else {
    // at least four rows per worker, so that its partial sums stay a small share of the traffic
    s.per_group = (int)std::min<int64_t>(std::max<int64_t>(most / groups, 1), (gate_rows + 3) / 4);
    s.workers = (int)(groups * s.per_group);
  }
  return s;
}

static int check_sizes(const char* what, int rows, int cols, int64_t gate_rows) {
  if (rows < 0 || cols <= 0) return fail(GPA_ERR_INVALID, "%s: bad sizes", what);
  if (cols % 8 || cols > 8192)
    return fail(GPA_ERR_UNSUPPORTED, "%s: cols must be a multiple of 8, at most 8192", what);
  if (rows > 0 && (gate_rows <= 0 || rows % gate_rows))
    return fail(GPA_ERR_INVALID, "%s: gate_rows must divide rows", what);
  return GPA_OK;
}

static bool dtype_ok(int d) { return d == GPA_DTYPE_F32 || d == GPA_DTYPE_BF16; }
static bool rows_ok(const void* p, int64_t stride) { return p && aligned16(p) && stride % 8 == 0; }
static bool kind_ok(int k) { return k == kNone || k == kLayer || k == kRms; }

template <typename TX, typename TY>
static int launch_fwd(const FwdParams& p, cudaStream_t st) {
  const int vec = p.cols / 8;
#define GPA_RN(V, W) fwd_kernel<V, W, TX, TY><<<(unsigned)(((int64_t)p.rows + 8 / W - 1) / (8 / W)), 256, 0, st>>>(p)
  if (vec <= 32) {
    GPA_RN(1, 1);
  } else if (vec <= 64) {
    GPA_RN(2, 1);
  } else if (vec > 256) {
    if (vec <= 512) GPA_RN(2, 8);
    else GPA_RN(4, 8);
  } else if constexpr (sizeof(TY) == 4) {   // few vectors per lane where a vector is many registers
    if (vec <= 128) GPA_RN(2, 2);
    else GPA_RN(2, 4);
  } else if (vec <= 128) {
    GPA_RN(4, 1);
  } else {
    if constexpr (sizeof(TX) == 2)
      if (p.post_kind == kNone) {   // layernorm's order of sums
        GPA_RN(8, 1);
        return check_launch("gpa_residual_norm");
      }
    GPA_RN(4, 2);   // or where it waits for many sums
  }
#undef GPA_RN
  return check_launch("gpa_residual_norm");
}

template <bool POST, typename TX, typename TY>
static int launch_bwd(const BwdParams& p, const Split& s, cudaStream_t st) {
#define GPA_RNB(W, V)                                                                  \
  {                                                                                    \
    constexpr int NG = W * 32 < 128 ? 128 / (W * 32) : 1;                              \
    bwd_kernel<POST, W, V, TX, TY><<<(s.workers + NG - 1) / NG, NG * W * 32, 0, st>>>(p); \
  }
  if (s.vpt == 2) GPA_RNB(16, 2)
  else if (s.wpr == 1) GPA_RNB(1, 1)
  else if (s.wpr == 2) GPA_RNB(2, 1)
  else if (s.wpr == 4) GPA_RNB(4, 1)
  else if (s.wpr == 8) GPA_RNB(8, 1)
  else GPA_RNB(16, 1)
#undef GPA_RNB
  return check_launch("gpa_residual_norm_backward");
}

}  // namespace resnorm
}  // namespace gpa

using namespace gpa;
using namespace gpa::resnorm;

extern "C" int gpa_residual_norm(const void* x, int x_dtype, int64_t x_stride, const void* y, int y_dtype,
                                 int64_t y_stride, const void* gate, int gate_dtype, int64_t gate_rows,
                                 int rows, int cols, int post_kind, const void* post_weight,
                                 const void* post_bias, float post_eps, int kind, const void* weight,
                                 const void* bias, int param_dtype, float eps, void* z, int64_t z_stride,
                                 void* h, int64_t h_stride, float* stats, void* stream) {
  const char* what = "gpa_residual_norm";
  if (!gate) gate_rows = rows;
  int rc = check_sizes(what, rows, cols, gate_rows);
  if (rc) return rc;
  if (!dtype_ok(x_dtype) || !dtype_ok(y_dtype) || !dtype_ok(gate_dtype) || !dtype_ok(param_dtype))
    return fail(GPA_ERR_INVALID, "%s: dtypes must be f32 or bf16", what);
  if (x_dtype == GPA_DTYPE_BF16 && y_dtype == GPA_DTYPE_F32)
    return fail(GPA_ERR_UNSUPPORTED, "%s: an f32 branch needs an f32 stream", what);
  if (!kind_ok(post_kind) || !kind_ok(kind)) return fail(GPA_ERR_INVALID, "%s: unknown norm kind", what);
  if (rows == 0) return ok();
  if (!rows_ok(x, x_stride) || !rows_ok(y, y_stride) || !rows_ok(z, z_stride) ||
      (kind != kNone && !rows_ok(h, h_stride)))
    return fail(GPA_ERR_INVALID, "%s: 16-byte aligned rows with strides that are multiples of 8 required", what);
  if (!aligned16(gate) || !aligned16(post_weight) || !aligned16(post_bias) || !aligned16(weight) ||
      !aligned16(bias) || !aligned16(stats))
    return fail(GPA_ERR_INVALID, "%s: gate, parameters and stats must be 16-byte aligned", what);
  const int pb = param_dtype == GPA_DTYPE_BF16;
  FwdParams p{x, y, z, h, x_stride, y_stride, z_stride, h_stride,
              {gate, gate_dtype == GPA_DTYPE_BF16}, gate_rows, rows, cols, post_kind, kind,
              {post_weight, pb}, {post_bias, pb}, {weight, pb}, {bias, pb}, post_eps, eps, stats};
  cudaStream_t st = (cudaStream_t)stream;
  if (x_dtype == GPA_DTYPE_BF16) return launch_fwd<__nv_bfloat16, __nv_bfloat16>(p, st);
  if (y_dtype == GPA_DTYPE_BF16) return launch_fwd<float, __nv_bfloat16>(p, st);
  return launch_fwd<float, float>(p, st);
}

extern "C" int64_t gpa_residual_norm_backward_workspace_bytes(int rows, int cols, int64_t gate_rows) {
  if (rows <= 0 || cols <= 0 || gate_rows <= 0 || rows % gate_rows) return 0;
  return (int64_t)split_rows(rows, cols, gate_rows).workers * kSlots * cols * 4;
}

extern "C" int gpa_residual_norm_backward(
    const void* dz, int64_t dz_stride, const void* dh, int64_t dh_stride, const void* z, int x_dtype,
    int64_t z_stride, const void* y, int y_dtype, int64_t y_stride, const float* stats, const void* gate,
    int gate_dtype, int64_t gate_rows, int rows, int cols, int post_kind, const void* post_weight,
    const void* post_bias, int kind, const void* weight, int param_dtype, void* dx, int64_t dx_stride,
    void* dy, int64_t dy_stride, void* dgate, void* dweight, void* dbias, void* dpost_weight,
    void* dpost_bias, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "gpa_residual_norm_backward";
  if (!gate) gate_rows = rows;
  int rc = check_sizes(what, rows, cols, gate_rows);
  if (rc) return rc;
  if (!dtype_ok(x_dtype) || !dtype_ok(y_dtype) || !dtype_ok(gate_dtype) || !dtype_ok(param_dtype))
    return fail(GPA_ERR_INVALID, "%s: dtypes must be f32 or bf16", what);
  if (x_dtype == GPA_DTYPE_BF16 && y_dtype == GPA_DTYPE_F32)
    return fail(GPA_ERR_UNSUPPORTED, "%s: an f32 branch needs an f32 stream", what);
  if (!kind_ok(post_kind) || !kind_ok(kind)) return fail(GPA_ERR_INVALID, "%s: unknown norm kind", what);
  if (rows == 0) return fail(GPA_ERR_INVALID, "%s: no rows (the gradients of the parameters are zero)", what);
  if (kind == kNone) dh = nullptr;
  if ((dz && !rows_ok(dz, dz_stride)) || (dh && !rows_ok(dh, dh_stride)) || !rows_ok(z, z_stride) ||
      !rows_ok(y, y_stride) || !rows_ok(dx, dx_stride) || !rows_ok(dy, dy_stride))
    return fail(GPA_ERR_INVALID, "%s: 16-byte aligned rows with strides that are multiples of 8 required", what);
  if (!stats || !aligned16(stats) || !aligned16(gate) || !aligned16(post_weight) || !aligned16(post_bias) ||
      !aligned16(weight) || !aligned16(dgate) || !workspace || !aligned16(workspace))
    return fail(GPA_ERR_INVALID, "%s: gate, parameters, stats and workspace must be 16-byte aligned", what);
  if (workspace_bytes < gpa_residual_norm_backward_workspace_bytes(rows, cols, gate_rows))
    return fail(GPA_ERR_INVALID, "%s: workspace too small", what);
  const Split s = split_rows(rows, cols, gate_rows);
  const int groups = (int)(rows / gate_rows);
  const int pbf = param_dtype == GPA_DTYPE_BF16, gbf = gate_dtype == GPA_DTYPE_BF16;
  const bool post = post_kind != kNone;
  if (!gate) dgate = nullptr;
  if (!post) dpost_weight = dpost_bias = nullptr;
  if (kind == kNone) dweight = dbias = nullptr;
  BwdParams p{dz, dh, z, y, dx, dy, dz_stride, dh_stride, z_stride, y_stride, dx_stride, dy_stride,
              {gate, gbf}, gate_rows, rows, cols, post_kind, kind, {post_weight, pbf}, {post_bias, pbf},
              {weight, pbf}, stats,
              {dgate != nullptr, dweight != nullptr, dbias != nullptr, dpost_weight != nullptr, dpost_bias != nullptr},
              s.whole, groups, s.per_group, s.workers, dgate, gbf, (float*)workspace};
  cudaStream_t st = (cudaStream_t)stream;
  if (x_dtype == GPA_DTYPE_BF16)
    rc = post ? launch_bwd<true, __nv_bfloat16, __nv_bfloat16>(p, s, st)
              : launch_bwd<false, __nv_bfloat16, __nv_bfloat16>(p, s, st);
  else if (y_dtype == GPA_DTYPE_BF16)
    rc = post ? launch_bwd<true, float, __nv_bfloat16>(p, s, st) : launch_bwd<false, float, __nv_bfloat16>(p, s, st);
  else
    rc = post ? launch_bwd<true, float, float>(p, s, st) : launch_bwd<false, float, float>(p, s, st);
  if (rc) return rc;
  void* gate_here = s.whole ? nullptr : dgate;
  if (!gate_here && !dweight && !dbias && !dpost_weight && !dpost_bias) return ok();
  SumParams q{(const float*)workspace, cols, s.workers, s.per_group, gate_here ? groups : 0,
              {gate_here, dweight, dbias, dpost_weight, dpost_bias}, {gbf, pbf, pbf, pbf, pbf}};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((cols + 31) / 32, 4 + q.gate_groups);
  cfg.blockDim = dim3(1024);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sum_kernel, q);
  if (e != cudaSuccess) return fail(GPA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}
