// The residual step around a block of a token model, one pass each way:
//
//   u = (h - mean_1) rstd_1      n = u * w1 (+ b1)      y = alpha x + g * n        the block's output h, normed, gated, added
//   t = (y - mean_2) rstd_2      z = t * w2 (+ b2)                                 the next block's normed input
//
// (root-mean-square norms: means 0).  Bound by bytes: 2 rows in and 2 out forward, 4 in and 2 out backward, so a row is read
// once, lives in registers between the two norms, and the weights are loaded once per block, which walks many rows.  y is
// rounded when it is stored; z and the backward are formed from the unrounded value (formed again from h and x, which costs
// the same bytes as reading y).  A row belongs to 1, 2, 4 or 8 waves by its width (at most 16 columns per lane).
//
// Backward:  a = dz w2,  D = dy + rstd_2 (a - mean(a) - t mean(a t)),  dx = alpha D,  c = D g w1,
//            dh = rstd_1 (c - mean(c) - u mean(c u)),   dw2 = sum dz t,  A = sum D u,  B = sum D  over a gate row's tokens,
//            dg = w1 A + b1 B,   dw1 = sum over gate rows of g A,   db1 of g B.
// Measured, bf16: 32768 x 4096 forward 199 us (5.4 TB/s), backward 352 (4.6, six rows of it); 16 x 1024 x 1024 36 and 39 us;
// 16 x 2048 5 us.  The next row's loads are in flight while a row is worked on (without: 271 and 899 us at 32768 x 4096).
// Column sums stay in registers over a block's rows, go through one fp32 partial per block and are folded in a fixed order.
#include <math.h>
#include "eovae_common.h"
#include "../../include/eovae_hip.h"

namespace {

typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));

struct NormArgs {
  const void *h, *x, *dy, *dz;
  void *y, *z, *dh, *dx;
  const void *w1, *b1, *w2, *b2, *gate;
  void *dw1, *db1, *dw2, *db2, *dgate;
  float *stats, *part;
  long long rows;
  int C, gates, layer, vec, p_f32, seg_rows, segs, group_units;
  long long per_gate;
  float alpha, eps;
};

__device__ __forceinline__ float ldp(const void* p, size_t i, int f32) { return f32 ? ((const float*)p)[i] : (float)((const __bf16*)p)[i]; }
__device__ __forceinline__ void stp(void* p, size_t i, int f32, float v) {
  if (f32) ((float*)p)[i] = v;
  else ((__bf16*)p)[i] = (__bf16)v;
}

template <int CTRL> __device__ __forceinline__ float dpp_add(float x) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_of(float x, int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l)); }
__device__ __forceinline__ float wsum(float v) {   // fixed order, every lane gets the sum (exchanges as in wave_sum_d)
  v = dpp_add<0xB1>(v);
  v = dpp_add<0x4E>(v);
  v = dpp_add<0x141>(v);
  v = dpp_add<0x140>(v);
  return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}

// sums of K values over the WPR waves of a row; `red` [2][K][waves of the block] alternates by parity: one barrier per call
template <int WPR, int K> __device__ __forceinline__ void row_sum(float (&v)[K], float* red, int& parity, int wave, int nwaves) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wsum(v[k]);
  if constexpr (WPR > 1) {
    float* r = red + parity * 2 * nwaves;
    parity ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) r[k * nwaves + wave] = v[k];
    __syncthreads();
    const int w0 = wave / WPR * WPR;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) s += r[k * nwaves + w0 + w];
      v[k] = s;
    }
  }
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// a lane's columns of a row: NV runs of eight, run i at (64 WPR i + lane) * 8
template <typename T, int WPR, int NV, bool VEC> struct Cols {
  static constexpr int N = NV * 8, RAW = NV * (int)sizeof(T) / 2;
  int l, C;                                   // VEC: rows and parameters can be read 16 bytes at a time (whole runs inside the row)
  __device__ __forceinline__ int col(int i) const { return (i * 64 * WPR + l) * 8; }
  __device__ __forceinline__ bool in(int i) const { return (VEC ? col(i / 8) : col(i / 8) + i % 8) < C; }
  struct Raw { u32x4 r[RAW]; };               // the row's bytes as they lie, requested one row ahead of their use
  __device__ __forceinline__ void request(Raw& o, const T* row) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = col(i);
      if constexpr (VEC) {
        const int at = c < C ? c : 0;           // behind the row: its head again, cleared by take()
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; ++k) o.r[i * (int)sizeof(T) / 2 + k] = *(const u32x4*)((const char*)(row + at) + 16 * k);
      } else if constexpr (sizeof(T) == 2) {
        bf16x8v v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = row[c + e < C ? c + e : 0];
        o.r[i] = __builtin_bit_cast(u32x4, v);
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          f32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = row[c + 4 * k + e < C ? c + 4 * k + e : 0];
          o.r[2 * i + k] = __builtin_bit_cast(u32x4, v);
        }
      }
    }
  }
  __device__ __forceinline__ void take(float (&o)[N], const Raw& w) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (sizeof(T) == 2) {
        const bf16x8v v = __builtin_bit_cast(bf16x8v, w.r[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[8 * i + e] = (float)v[e];
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const f32x4 v = __builtin_bit_cast(f32x4, w.r[2 * i + k]);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[8 * i + 4 * k + e] = v[e];
        }
      }
      if constexpr (VEC) {
        if (col(i) >= C)
#pragma unroll
          for (int e = 0; e < 8; ++e) o[8 * i + e] = 0.f;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!in(8 * i + e)) o[8 * i + e] = 0.f;
      }
    }
  }
  __device__ __forceinline__ void store(const float (&o)[N], T* row) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = col(i);
      if constexpr (VEC) {
        if (c < C) {
          if constexpr (sizeof(T) == 2) {
            bf16x8v v;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (__bf16)o[8 * i + e];
            *(bf16x8v*)(row + c) = v;
          } else {
            *(f32x4*)(row + c) = f32x4{o[8 * i], o[8 * i + 1], o[8 * i + 2], o[8 * i + 3]};
            *(f32x4*)(row + c + 4) = f32x4{o[8 * i + 4], o[8 * i + 5], o[8 * i + 6], o[8 * i + 7]};
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < C) row[c + e] = (T)o[8 * i + e];
      }
    }
  }
  __device__ __forceinline__ void store_param(const float (&o)[N], void* p, size_t off, int f32) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = col(i);
      if constexpr (VEC) {
        if (c < C) {
          if (f32) {
            *(f32x4*)((float*)p + off + c) = f32x4{o[8 * i], o[8 * i + 1], o[8 * i + 2], o[8 * i + 3]};
            *(f32x4*)((float*)p + off + c + 4) = f32x4{o[8 * i + 4], o[8 * i + 5], o[8 * i + 6], o[8 * i + 7]};
          } else {
            bf16x8v v;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (__bf16)o[8 * i + e];
            *(bf16x8v*)((__bf16*)p + off + c) = v;
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < C) stp(p, off + c + e, f32, o[8 * i + e]);
      }
    }
  }
  // a parameter row of either type; absent: `none` everywhere inside the row, 0 behind it
  __device__ __forceinline__ void param(float (&o)[N], const void* p, size_t off, int f32, float none) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = col(i);
      if (!p) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[8 * i + e] = c + e < C ? none : 0.f;
      } else if constexpr (VEC) {
        const size_t at = off + (c < C ? c : 0);
        if (f32) {
          const f32x4 x = *(const f32x4*)((const float*)p + at), y = *(const f32x4*)((const float*)p + at + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[8 * i + e] = x[e], o[8 * i + 4 + e] = y[e];
        } else {
          const bf16x8v v = *(const bf16x8v*)((const __bf16*)p + at);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[8 * i + e] = (float)v[e];
        }
        if (c >= C)
#pragma unroll
          for (int e = 0; e < 8; ++e) o[8 * i + e] = 0.f;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[8 * i + e] = c + e < C ? ldp(p, off + c + e, f32) : 0.f;
      }
    }
  }
};

template <typename T, int WPR, int NV, bool LAYER, bool VEC>
__global__ __launch_bounds__(WPR == 8 ? 512 : 256) void norm_fwd_kernel(const NormArgs a) {
  constexpr int N = NV * 8, WAVES = WPR == 8 ? 8 : 4, SLOTS = WAVES / WPR;
  __shared__ float red[2 * 2 * WAVES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slot = wave / WPR;
  const Cols<T, WPR, NV, VEC> cs{(int)(threadIdx.x % (64 * WPR)), a.C};
  int parity = 0;
  float w1[N], w2[N], g[N], b1[LAYER ? N : 1], b2[LAYER ? N : 1];
  cs.param(w1, a.w1, 0, a.p_f32, 1.f);
  cs.param(w2, a.w2, 0, a.p_f32, 1.f);
  if constexpr (LAYER) {
    cs.param(b1, a.b1, 0, a.p_f32, 0.f);
    cs.param(b2, a.b2, 0, a.p_f32, 0.f);
  }
  const float n = (float)a.C;       // divided by, not multiplied with 1 / n: the mean of equal values is that value
  long long until = 0;                                          // rows below it use the gate row in g
  typename Cols<T, WPR, NV, VEC>::Raw rh, rx;
  const long long step = (long long)gridDim.x * SLOTS;
  const auto row_of = [&](long long r0) { return r0 + slot < a.rows ? r0 + slot : a.rows - 1; };   // an idle slot repeats a row and stores nothing
  const auto request = [&](long long r0) {
    cs.request(rh, (const T*)a.h + row_of(r0) * a.C);
    cs.request(rx, (const T*)a.x + row_of(r0) * a.C);
  };
  request((long long)blockIdx.x * SLOTS);
  for (long long r0 = (long long)blockIdx.x * SLOTS; r0 < a.rows; r0 += step) {
    const bool on = r0 + slot < a.rows;
    const long long row = row_of(r0);
    float h[N], x[N];
    cs.take(h, rh);
    cs.take(x, rx);
    if (r0 + step < a.rows) request(r0 + step);
    if (row >= until) {
      const long long gr = a.gates ? row / a.per_gate : 0;
      cs.param(g, a.gate, (size_t)gr * a.C, a.p_f32, 1.f);
      until = a.gates ? (gr + 1) * a.per_gate : a.rows;
    }
    float m1 = 0.f, m2 = 0.f, s[1];
    if (LAYER) {
      s[0] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) s[0] += h[i];
      row_sum<WPR, 1>(s, red, parity, wave, WAVES);
      m1 = s[0] / n;
    }
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (LAYER) h[i] = cs.in(i) ? h[i] - m1 : 0.f;
      s[0] += h[i] * h[i];
    }
    row_sum<WPR, 1>(s, red, parity, wave, WAVES);
    const float r1 = 1.f / sqrtf(s[0] / n + a.eps);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = a.alpha * x[i] + g[i] * (LAYER ? h[i] * r1 * w1[i] + b1[LAYER ? i : 0] : h[i] * r1 * w1[i]);
    if (on) cs.store(x, (T*)a.y + row * a.C);
    float r2 = 0.f;
    if (a.z) {
      if (LAYER) {
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) s[0] += x[i];
        row_sum<WPR, 1>(s, red, parity, wave, WAVES);
        m2 = s[0] / n;
      }
      s[0] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if constexpr (LAYER) x[i] = cs.in(i) ? x[i] - m2 : 0.f;
        s[0] += x[i] * x[i];
      }
      row_sum<WPR, 1>(s, red, parity, wave, WAVES);
      r2 = 1.f / sqrtf(s[0] / n + a.eps);
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = LAYER ? x[i] * r2 * w2[i] + b2[LAYER ? i : 0] : x[i] * r2 * w2[i];
      if (on) cs.store(x, (T*)a.z + row * a.C);
    }
    if (a.stats && on && threadIdx.x % (64 * WPR) == 0) *(f32x4*)(a.stats + 4 * row) = f32x4{m1, r1, m2, r2};
  }
}

// A block's unit of rows lies inside one gate row (segs units to each), or is group_units whole gate rows.
// part: [units][parts][C], parts: dw1, dw2, then db1, db2 (layer norms), then the gate row's dg when segs > 1
// The next row's bytes are requested before this row is worked on (AHEAD), except where the registers do not allow it.
template <typename T, int WPR, int NV, bool LAYER, bool VEC>
__global__ __launch_bounds__(WPR == 8 ? 512 : 256) void norm_bwd_kernel(const NormArgs a) {
  constexpr int N = NV * 8, WAVES = WPR == 8 ? 8 : 4, SLOTS = WAVES / WPR, LANES = 64 * WPR, PARTS = LAYER ? 5 : 3;
  constexpr bool AHEAD = WPR < 8;
  __shared__ float red[2 * 2 * WAVES];
  __shared__ __attribute__((aligned(16))) float fold[SLOTS > 1 ? (SLOTS - 1) * LANES * (N + 4) : 1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slot = wave / WPR;
  const Cols<T, WPR, NV, VEC> cs{(int)(threadIdx.x % LANES), a.C};
  int parity = 0;
  float w1[N], w2[N], b1[LAYER ? N : 1], g[N];
  // layer norms of the widest rows: the sums (of this thread's own columns) live in LDS, 512 threads leave 256 registers each
  constexpr bool SIDE = WPR == 8 && LAYER;
  __shared__ float side[SIDE ? 4 : 1][SIDE ? N : 1][SIDE ? 512 : 1];
  float sA[SIDE ? 1 : N], sW2[SIDE ? 1 : N], sB[LAYER && !SIDE ? N : 1], sB2[LAYER && !SIDE ? N : 1];
  cs.param(w1, a.w1, 0, a.p_f32, 1.f);
  if constexpr (LAYER) cs.param(b1, a.b1, 0, a.p_f32, 0.f);
  cs.param(w2, a.w2, 0, a.p_f32, 1.f);
  const auto clear = [&](auto& v) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
  };
  const auto clear_ab = [&]() {
    if constexpr (SIDE) {
#pragma unroll
      for (int i = 0; i < N; ++i) side[0][i][threadIdx.x] = side[2][i][threadIdx.x] = 0.f;
    } else {
      clear(sA);
      if constexpr (LAYER) clear(sB);
    }
  };
  clear_ab();
  if constexpr (SIDE) {
#pragma unroll
    for (int i = 0; i < N; ++i) side[1][i][threadIdx.x] = side[3][i][threadIdx.x] = 0.f;
  } else {
    clear(sW2);
    if constexpr (LAYER) clear(sB2);
  }
  const float n = (float)a.C;       // divided by, not multiplied with 1 / n: the mean of equal values is that value
  const long long gates = a.gates ? a.gates : 1;
  const bool single = a.per_gate == 1 && a.gates;              // a gate row per token: its gradient leaves with the token
  // sums of a value over the block's slots, in slot order, in slot 0 (all threads call)
  const auto join = [&](float (&v)[N]) {
    if constexpr (SLOTS > 1) {
      __syncthreads();
      if (slot > 0)
#pragma unroll
        for (int i = 0; i < N; i += 4) *(f32x4*)(fold + ((slot - 1) * LANES + cs.l) * (N + 4) + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
      __syncthreads();
      if (slot == 0)
        for (int s = 0; s < SLOTS - 1; ++s)
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] += fold[(s * LANES + cs.l) * (N + 4) + i];
    }
  };
  const long long unit = blockIdx.x;
  float* part = a.part + (size_t)unit * PARTS * a.C;
  // slot 0: v (times the gate row, for `gated`) into part `which`; `more`: onto what an earlier gate row of this unit left there
  const auto keep = [&](const float (&v)[N], int which, bool gated, bool more) {
    if (slot == 0)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (cs.in(i)) {
          float* at = part + (size_t)which * a.C + cs.col(i / 8) + i % 8;
          const float x = gated ? g[i] * v[i] : v[i];
          *at = more ? *at + x : x;
        }
  };
  long long g0, g1, ra, rb;                                    // gate rows [g0, g1), tokens [ra, rb) of each
  if (a.segs > 0) {
    g0 = unit / a.segs;
    g1 = g0 + 1;
    ra = unit % a.segs * a.seg_rows;
    rb = ra + a.seg_rows < a.per_gate ? ra + a.seg_rows : a.per_gate;
  } else {
    g0 = unit * a.group_units;
    g1 = g0 + a.group_units < gates ? g0 + a.group_units : gates;
    ra = 0;
    rb = a.per_gate;
  }
  typename Cols<T, WPR, NV, VEC>::Raw rh, rx, rd, rq;
  f32x4 rs;
  for (long long gr = g0; gr < (single ? g0 + 1 : g1); ++gr) {
    if (!single) cs.param(g, a.gate, (size_t)gr * a.C, a.p_f32, 1.f);
    const long long lo = single ? 0 : ra, hi = single ? g1 - g0 : rb, base = single ? g0 : gr * a.per_gate;
    const auto row_of = [&](long long r0) { return base + (r0 + slot < hi ? r0 + slot : hi - 1); };
    const auto request = [&](long long r0) {
      const long long at = row_of(r0) * a.C;
      cs.request(rh, (const T*)a.h + at);
      cs.request(rx, (const T*)a.x + at);
      cs.request(rd, (const T*)a.dy + at);
      if (a.dz) cs.request(rq, (const T*)a.dz + at);
      rs = *(const f32x4*)(a.stats + 4 * row_of(r0));
    };
    if (AHEAD) request(lo);
    for (long long r0 = lo; r0 < hi; r0 += SLOTS) {
      const bool on = r0 + slot < hi;
      const long long row = row_of(r0);
      if (!AHEAD) request(r0);
      if (single) cs.param(g, a.gate, (size_t)row * a.C, a.p_f32, 1.f);
      float h[N], y[N], d[N], q[N];
      cs.take(h, rh);
      cs.take(y, rx);
      cs.take(d, rd);
      if (a.dz) cs.take(q, rq);
      const f32x4 st = rs;
      if (AHEAD && r0 + SLOTS < hi) request(r0 + SLOTS);
      // columns behind the row are zero everywhere (a layer norm's mean has to be kept out of them)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        h[i] = (h[i] - (LAYER ? st[0] : 0.f)) * st[1];
        if (LAYER && !cs.in(i)) h[i] = 0.f;
      }
      if (a.dz) {
        float s[LAYER ? 2 : 1] = {};
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float t = a.alpha * y[i] + g[i] * (LAYER ? h[i] * w1[i] + b1[LAYER ? i : 0] : h[i] * w1[i]);
          y[i] = (t - (LAYER ? st[2] : 0.f)) * st[3];
          if (LAYER && !cs.in(i)) y[i] = 0.f;
          const float e = q[i] * w2[i];
          s[0] += e * y[i];
          if constexpr (LAYER) s[1] += e;
          if (on) {
            if constexpr (SIDE) side[3][i][threadIdx.x] += q[i] * y[i];
            else sW2[i] += q[i] * y[i];
            if constexpr (SIDE) side[1][i][threadIdx.x] += q[i];
            else if constexpr (LAYER) sB2[i] += q[i];
          }
          q[i] = e;
        }
        row_sum<WPR, LAYER ? 2 : 1>(s, red, parity, wave, WAVES);
        const float mt = s[0] / n, ma = LAYER ? s[LAYER ? 1 : 0] / n : 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          d[i] += st[3] * (LAYER ? q[i] - ma - y[i] * mt : q[i] - y[i] * mt);
          if (LAYER && !cs.in(i)) d[i] = 0.f;
        }
      }
      float s[LAYER ? 2 : 1] = {};
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float e = d[i] * g[i], c = e * w1[i];
        s[0] += c * h[i];
        if constexpr (LAYER) s[1] += c;
        y[i] = a.alpha * d[i];
        q[i] = c;
        if (on) {
          if constexpr (SIDE) side[2][i][threadIdx.x] += (single ? e : d[i]) * h[i];
          else sA[i] += (single ? e : d[i]) * h[i];
          if constexpr (SIDE) side[0][i][threadIdx.x] += single ? e : d[i];
          else if constexpr (LAYER) sB[i] += single ? e : d[i];
        }
      }
      if (on) cs.store(y, (T*)a.dx + row * a.C);
      row_sum<WPR, LAYER ? 2 : 1>(s, red, parity, wave, WAVES);
      const float mu = s[0] / n, mc = LAYER ? s[LAYER ? 1 : 0] / n : 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = st[1] * (LAYER ? q[i] - mc - h[i] * mu : q[i] - h[i] * mu);
      if (on) cs.store(y, (T*)a.dh + row * a.C);
      if (single && on && a.dgate) {
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = d[i] * (LAYER ? h[i] * w1[i] + b1[LAYER ? i : 0] : h[i] * w1[i]);
        cs.store_param(y, a.dgate, (size_t)row * a.C, a.p_f32);
      }
    }
    float u[N], v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = SIDE ? side[SIDE ? 2 : 0][SIDE ? i : 0][SIDE ? threadIdx.x : 0] : sA[SIDE ? 0 : i];
    join(u);
    keep(u, 0, !single, gr > g0);
    if constexpr (LAYER) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = SIDE ? side[0][SIDE ? i : 0][SIDE ? threadIdx.x : 0] : sB[SIDE ? 0 : i];
      join(v);
      keep(v, 2, !single, gr > g0);
    }
    if (!single) {
      if (slot == 0 && a.dgate) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = LAYER ? w1[i] * u[i] + b1[LAYER ? i : 0] * v[i] : w1[i] * u[i];
        if (a.segs > 1) keep(v, PARTS - 1, false, false);
        else cs.store_param(v, a.dgate, (size_t)gr * a.C, a.p_f32);
      }
      clear_ab();
    }
  }
  float v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = SIDE ? side[SIDE ? 3 : 0][SIDE ? i : 0][SIDE ? threadIdx.x : 0] : sW2[SIDE ? 0 : i];
  join(v);
  keep(v, 1, false, false);
  if constexpr (LAYER) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = SIDE ? side[SIDE ? 1 : 0][SIDE ? i : 0][SIDE ? threadIdx.x : 0] : sB2[SIDE ? 0 : i];
    join(v);
    keep(v, 3, false, false);
  }
}

// 64 columns x 16 runs of partials per block, each run in order, the runs in order
__global__ __launch_bounds__(1024) void norm_fold_kernel(const NormArgs a, int units, int nweights) {
  __shared__ float s[16][65];
  const int parts = a.layer ? 5 : 3, cb = (a.C + 63) / 64;
  const int out = blockIdx.x / cb, c = (int)(blockIdx.x % cb) * 64 + (threadIdx.x & 63), run = threadIdx.x >> 6;
  int which, u0, n;
  if (out < nweights) {
    which = out;
    u0 = 0;
    n = units;
  } else {
    which = parts - 1;
    u0 = (out - nweights) * a.segs;
    n = a.segs;
  }
  const int len = (n + 15) / 16, lo = run * len, hi = min(n, lo + len);
  float sum = 0.f;
  if (c < a.C)
#pragma unroll 8
    for (int u = lo; u < hi; ++u) sum += a.part[((size_t)(u0 + u) * parts + which) * a.C + c];
  s[run][threadIdx.x & 63] = sum;
  __syncthreads();
  if (run || c >= a.C) return;
  float v = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) v += s[r][threadIdx.x];
  if (out < nweights) {
    void* p = which == 0 ? a.dw1 : which == 1 ? a.dw2 : which == 2 ? a.db1 : a.db2;
    if (p) stp(p, c, a.p_f32, v);
  } else {
    stp(a.dgate, (size_t)(out - nweights) * a.C + c, a.p_f32, v);
  }
}

constexpr int UNITS = 512;          // blocks of a long backward: two per CU

// rows of a unit and how units meet gate rows
void plan(const eovae_token_norm* d, NormArgs& a, long long& units) {
  const long long gates = d->gates ? d->gates : 1;
  a.per_gate = d->rows / gates;
  const int slots = d->channels <= 1024 ? 4 : d->channels <= 2048 ? 2 : 1;
  long long want = (d->rows + UNITS - 1) / UNITS;                     // rows per unit
  want = (want + slots - 1) / slots * slots;
  if (a.per_gate >= want) {
    a.segs = (int)((a.per_gate + want - 1) / want);
    const long long even = (a.per_gate + a.segs - 1) / a.segs;
    a.seg_rows = (int)((even + slots - 1) / slots * slots);
    a.segs = (int)((a.per_gate + a.seg_rows - 1) / a.seg_rows);
    a.group_units = 0;
    units = gates * a.segs;
  } else {
    a.segs = 0;
    a.seg_rows = 0;
    a.group_units = (int)(want / a.per_gate);
    units = (gates + a.group_units - 1) / a.group_units;
  }
}

enum { FORWARD, BACKWARD, SIZES };      // SIZES: shapes and types only
int check(const eovae_token_norm* d, const char* who, int mode) {
  EOVAE_CHECK_ARG(d != nullptr, "%s: null descriptor", who);
  EOVAE_CHECK_ARG(d->dtype == EOVAE_F32 || d->dtype == EOVAE_BF16, "%s: dtype %d (0 fp32, 1 bf16)", who, d->dtype);
  EOVAE_CHECK_ARG(d->param_dtype == EOVAE_F32 || d->param_dtype == EOVAE_BF16, "%s: param dtype %d (0 fp32, 1 bf16)", who, d->param_dtype);
  EOVAE_CHECK_ARG(d->rows >= 1 && d->rows <= (1ll << 38) && d->channels >= 1 && d->channels <= 8192, "%s: %lld rows of %d channels (1 .. 8192)", who,
                  d->rows, d->channels);
  EOVAE_CHECK_ARG(d->gates >= 0 && d->gates <= (1ll << 30) && (d->gates == 0 || d->rows % d->gates == 0), "%s: %lld gate rows for %lld rows", who, d->gates,
                  d->rows);
  if (mode == SIZES) return EOVAE_OK;
  EOVAE_CHECK_ARG((d->gates > 0) == (d->gate != nullptr), "%s: gate and gates disagree", who);
  EOVAE_CHECK_ARG(d->h && d->x && d->w1, "%s: null h, x or w1", who);
  EOVAE_CHECK_ARG(d->layer || (!d->b1 && !d->b2), "%s: a root-mean-square norm has no bias", who);
  EOVAE_CHECK_ARG(isfinite(d->alpha) && d->eps > 0.f && isfinite(d->eps), "%s: alpha or eps", who);
  if (mode == BACKWARD) {
    EOVAE_CHECK_ARG(d->dy && d->dh && d->dx && d->stats, "%s: null dy, dh, dx or stats", who);
    EOVAE_CHECK_ARG(!d->dz || d->w2, "%s: dz without w2", who);
    EOVAE_CHECK_ARG(!d->dgate || d->gate, "%s: dgate without a gate", who);
  } else {
    EOVAE_CHECK_ARG(d->y && (!d->z || d->w2), "%s: null y, or z without w2", who);
  }
  return EOVAE_OK;
}

NormArgs args_of(const eovae_token_norm* d) {
  NormArgs a{};
  a.h = d->h; a.x = d->x; a.dy = d->dy; a.dz = d->dz;
  a.y = d->y; a.z = d->z; a.dh = d->dh; a.dx = d->dx;
  a.w1 = d->w1; a.b1 = d->b1; a.w2 = d->w2; a.b2 = d->b2; a.gate = d->gate;
  a.dw1 = d->dw1; a.db1 = d->db1; a.dw2 = d->dw2; a.db2 = d->db2; a.dgate = d->dgate;
  a.stats = d->stats;
  a.rows = d->rows; a.C = d->channels; a.gates = (int)d->gates; a.layer = d->layer ? 1 : 0;
  a.p_f32 = d->param_dtype == EOVAE_F32;
  a.alpha = d->alpha; a.eps = d->eps;
  const void* ptrs[] = {d->h, d->x, d->dy, d->dz, d->y, d->z, d->dh, d->dx, d->w1, d->b1, d->w2, d->b2, d->gate, d->dgate};
  bool vec = d->channels % 8 == 0;
  for (const void* p : ptrs) vec = vec && (size_t)p % 16 == 0;
  a.vec = vec;
  return a;
}

// waves per row and vectors per lane by the row's width
#define NORM_WIDTHS(T, KERNEL, LAYER, VEC, blocks, st, a)                                                          \
  do {                                                                                                              \
    if ((a).C <= 512) hipLaunchKernelGGL((KERNEL<T, 1, 1, LAYER, VEC>), dim3(blocks), dim3(256), 0, st, a);          \
    else if ((a).C <= 1024) hipLaunchKernelGGL((KERNEL<T, 1, 2, LAYER, VEC>), dim3(blocks), dim3(256), 0, st, a);    \
    else if ((a).C <= 2048) hipLaunchKernelGGL((KERNEL<T, 2, 2, LAYER, VEC>), dim3(blocks), dim3(256), 0, st, a);    \
    else if ((a).C <= 4096) hipLaunchKernelGGL((KERNEL<T, 4, 2, LAYER, VEC>), dim3(blocks), dim3(256), 0, st, a);    \
    else hipLaunchKernelGGL((KERNEL<T, 8, 2, LAYER, VEC>), dim3(blocks), dim3(512), 0, st, a);                      \
  } while (0)
#define NORM_TYPES(T, KERNEL, blocks, st, a)                                        \
  do {                                                                              \
    if ((a).layer && (a).vec) NORM_WIDTHS(T, KERNEL, true, true, blocks, st, a);     \
    else if ((a).layer) NORM_WIDTHS(T, KERNEL, true, false, blocks, st, a);          \
    else if ((a).vec) NORM_WIDTHS(T, KERNEL, false, true, blocks, st, a);            \
    else NORM_WIDTHS(T, KERNEL, false, false, blocks, st, a);                        \
  } while (0)
#define NORM_DISPATCH(KERNEL, f32, blocks, st, a)              \
  do {                                                         \
    if (f32) NORM_TYPES(float, KERNEL, blocks, st, a);          \
    else NORM_TYPES(__bf16, KERNEL, blocks, st, a);             \
  } while (0)

}  // namespace

extern "C" {
size_t eovae_token_norm_workspace(const eovae_token_norm* d) {
  if (check(d, "token_norm_workspace", SIZES)) return 0;
  NormArgs a = args_of(d);
  long long units;
  plan(d, a, units);
  return (size_t)units * (a.layer ? 5 : 3) * a.C * 4;
}

int eovae_token_norm_fwd(const eovae_token_norm* d, void* stream) {
  const int rc = check(d, "token_norm_fwd", FORWARD);
  if (rc) return rc;
  NormArgs a = args_of(d);
  a.per_gate = d->gates ? d->rows / d->gates : 1;
  const int slots = a.C <= 1024 ? 4 : a.C <= 2048 ? 2 : 1;
  long long blocks = (a.rows + slots - 1) / slots;
  if (blocks > 2048) blocks = 2048;
  NORM_DISPATCH(norm_fwd_kernel, d->dtype == EOVAE_F32, (unsigned)blocks, (hipStream_t)stream, a);
  EOVAE_CHECK_LAUNCH("token_norm_fwd");
  return EOVAE_OK;
}

int eovae_token_norm_bwd(const eovae_token_norm* d, void* stream) {
  const int rc = check(d, "token_norm_bwd", BACKWARD);
  if (rc) return rc;
  NormArgs a = args_of(d);
  long long units;
  plan(d, a, units);
  const size_t need = (size_t)units * (a.layer ? 5 : 3) * a.C * 4;
  EOVAE_CHECK_ARG(d->ws && (size_t)d->ws % 16 == 0 && d->ws_bytes >= need, "token_norm_bwd: workspace of %zu bytes, needs %zu (16-byte aligned)",
                  d->ws_bytes, need);
  a.part = (float*)d->ws;
  NORM_DISPATCH(norm_bwd_kernel, d->dtype == EOVAE_F32, (unsigned)units, (hipStream_t)stream, a);
  EOVAE_CHECK_LAUNCH("token_norm_bwd");
  const int nweights = a.layer ? 4 : 2, cb = (a.C + 63) / 64;
  const long long gates = a.segs > 1 && a.dgate ? a.gates : 0;
  hipLaunchKernelGGL(norm_fold_kernel, dim3((unsigned)((nweights + gates) * cb)), dim3(1024), 0, (hipStream_t)stream, a, (int)units, nweights);
  EOVAE_CHECK_LAUNCH("token_norm_bwd");
  return EOVAE_OK;
}
}
