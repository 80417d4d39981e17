// Backward of the token attention (token_attn_common.h), without float atomics: two passes that each own their outputs.
//
//   P_m  = exp2(S_m - lse_m)            dA = dO V^T            w = (1, -lambda)
//   dS_m = P_m o (w_m dA - delta_m)     delta_m = w_m sum_d dO o O_m
//   dQ_m = scale dS_m K_m    dK_m = scale dS_m^T Q_m    dV = (sum_m w_m P_m)^T dO
//   dbias[bucket] = sum of dS_0 (+ dS_1) over its pairs       dlambda = - sum dO o O_1
//
// delta comes from stored outputs, rounded to the tensors' type: good for dQ, whose sum it enters with the mean of K only (the row's
// own sum P dA is known when the pass is over: dK/dV takes that one where it is formed), but not for the two sums that it could
// drown.  The last buckets hold nearly all of a long row's probability, and
// there sum dS = w (sum P dA - (mean of dA over the WHOLE row) (sum P)) is a difference of large values; lambda's gradient is
// that mean.  Both are formed in fp32 from P and dA themselves, row by row; the mean is divided by the row's own sum of P, so that
// a common error of P's scale (lse's rounding) cancels.
//
// attn_dq: a wave owns 32 queries and walks the keys; it also forms delta from O (for the second pass), the bias gradient's
// partial sums (pairs of one distance lie on a diagonal of the score tile) and lambda's.  attn_dkv: a wave owns 32 keys and
// walks the queries of every head that shares its key head, so shared heads' gradients are summed in a fixed order.  The
// scores are formed in both passes (7 products instead of 5): the price of bit-reproducible gradients without a
// [queries][keys] buffer.  Bound by vector instructions (exp2, the gradients' two operations per score, conversions) beside the
// matrix pipes.  bf16, measured: 16 x 8 heads x 1024 x 64 dQ 82 us (630 TFLOP/s of its three products), 110 .. 119 with the bias
// gradient, dK/dV 105 .. 112 (620 of four); 4 x 8 x 2048 x 128 dQ 127 us (810), dK/dV 201 (680); two maps of the same size 162 and 301.
// No kernel here may spill: hipcc 7.2 has brought a value spilled half to registers, half to scratch back with a register missing.
#include <math.h>
#include <type_traits>
#include "token_attn_common.h"

using namespace tok;

namespace {

// a wave's score gradients by diagonal: 64 rows (63 distances) of 32 queries, 4 floats apart from the next row's banks
constexpr int SCR = 36, SCR_FLOATS = 64 * SCR;

// fp32's matrix instructions are 16 times slower than bf16's: with fewer blocks of 128 rows than the chip has CUs, a call is a
// handful of long chains of them.  SPLIT (fp32 only): a block owns 32 rows, its four waves share the other side's tiles and add
// up through LDS at the end, and the tiles' fragments come from memory (their loads hide behind the matrix instructions), so that
// LDS is free for the sums.
template <int D> constexpr int meet_bytes() { return 4 * 32 * (D + 4) * 4; }

// the four waves' [32 columns of acc][D] tiles, added in wave order and stored as rows row0 + column < limit
template <typename T, int D>
__device__ __forceinline__ void meet_sum(float* meet, const f32x16 (&acc)[D / 32], float scale, T* out, long long ld, int row0, int limit, int wave,
                                         int lane) {
  constexpr int MROW = D + 4;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *(f32x4*)(meet + (wave * 32 + (lane & 31)) * MROW + 32 * j + 8 * g + 4 * (lane >> 5)) =
          f32x4{acc[j][4 * g], acc[j][4 * g + 1], acc[j][4 * g + 2], acc[j][4 * g + 3]};
  __syncthreads();
  for (int i = 64 * wave + lane; i < 32 * D / 4; i += 256) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    if (row0 + r >= limit) break;
    f32x4 v = *(const f32x4*)(meet + r * MROW + d);
#pragma unroll
    for (int w = 1; w < 4; ++w) v += *(const f32x4*)(meet + (w * 32 + r) * MROW + d);
    store4(out + (long long)(row0 + r) * ld + d, scale * v[0], scale * v[1], scale * v[2], scale * v[3]);
  }
}

template <typename T, int D, int MAPS, bool SPLIT>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attn_dq_kernel(const Params p) {
  using TK = Tile<T, D>;
  constexpr int W = D / MAPS;
  constexpr int NT = !SPLIT && D <= 64 && TK::ROWS == 64 ? 2 : 1, RB = SPLIT ? 32 : 128;           // 32-key tiles worked on together, as the registers allow
  extern __shared__ __attribute__((aligned(16))) char lds[];
  float* tab = (float*)(lds + (SPLIT ? meet_bytes<D>() : (int)Stream<T, D>::BYTES));
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int ntab = p.bk.n ? 2 * (p.bk.reach + PAD) + 1 : 0, reach = p.bk.reach;
  float* diag = tab + ntab + wave * ntab;                        // [4][ntab]: sums of score gradients by distance
  float* scr = tab + 5 * ntab + 3 - (5 * ntab + 3) % 4 + wave * SCR_FLOATS;
  const int nbh = p.B * p.H, tiles = (p.Sq + RB - 1) / RB;
  const int tile = tiles - 1 - (int)blockIdx.x / nbh;
  int b, hk, h;
  split_bh(p, (int)blockIdx.x % nbh, b, hk, h);
  const int row0 = tile * RB, wrow = SPLIT ? 0 : 32 * wave, start = uniform(start_of(p, b));
  const int rlast = min(row0 + RB, p.Sq) - 1;
  int kend = uniform(key_limit(p, b));
  if (p.causal) kend = min(kend, start + rlast + 1);
  const int qrow = row0 + wrow + (lane & 31);
  const bool live = qrow < p.Sq;
  const int qlo = start + row0 + wrow, qhi = qlo + 31, qpos = start + qrow;
  const T* kb = (const T*)p.k + b * p.kb + hk * p.kh;
  const T* vb = (const T*)p.v + b * p.vb + hk * p.vh;
  const T* qp = (const T*)p.q + b * p.qb + h * p.qh + (long long)qrow * p.qs;
  const size_t orow = (((size_t)b * p.Sq + qrow) * p.H + h) * D;
  Frag<T> qf[D / 16], gf[D / 16];
  float lam = 0.f, d1 = 0.f, d2 = 0.f;
  if constexpr (MAPS == 2) lam = ldf(p.lam, h, p.lam_f32);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    qf[i] = frag_global(qp, i, lane, live);
    gf[i] = frag_global((const T*)p.d_o + orow, i, lane, live);
    const Frag<T> of = frag_global((const T*)p.o + orow, i, lane, live);
    if constexpr (MAPS == 2) {
      const Frag<T> o2 = frag_global((const T*)p.o2 + orow, i, lane, live);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        d1 += (float)gf[i].x[e] * ((float)of.x[e] + lam * (float)o2.x[e]);
        d2 += (float)gf[i].x[e] * (float)o2.x[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) d1 += (float)gf[i].x[e] * (float)of.x[e];
    }
  }
  d1 = column_sum(d1);
  d2 = column_sum(d2);
  const bool sums = p.part || p.lam_part;                          // sum P dA is formed anyway
  float lse[MAPS], delta[MAPS];
  delta[0] = d1;
  if constexpr (MAPS == 2) delta[1] = -lam * d2;
#pragma unroll
  for (int a = 0; a < MAPS; ++a) {
    const size_t at = (((size_t)b * p.H + h) * MAPS + a) * p.Sq + qrow;
    lse[a] = live ? p.lse[at] : INFINITY;
    if (!sums && live && half == 0 && (!SPLIT || wave == 0)) p.delta[at] = delta[a];
  }
  float base = 0.f;
  bool wide = false;
  if (p.bk.n) {
    fill_bias(p, tab, h, tid, 256, false);                             // does not wait for what is hardly ever so
    wide = wide_head(p, h, lane);
    if (wide) {
      fill_bias(p, tab, h, tid, 256, true);
      base = row_base(p, h, qpos, kend);
    }
    if (tid == 0 && b == 0 && tile == 0) p.wide[h] = wide;
    if (wide && live && half == 0 && (!SPLIT || wave == 0)) p.base[((size_t)b * p.H + h) * p.Sq + qrow] = base;
    if (p.part) {
      for (int i = lane; i < ntab; i += 64) diag[i] = 0.f;
      for (int i = lane; i < SCR_FLOATS; i += 64) scr[i] = 0.f;
    }
    if constexpr (SPLIT) __syncthreads();      // the table is every thread's work; the streamed form's first barrier is its first tile's
  }
  f32x16 acc[D / 32];
#pragma unroll
  for (int j = 0; j < D / 32; ++j) acc[j] = zero16();
  const float c = positive_scale(p.scale, qf);
  // of this lane's query and map: sum P dA and sum P over the row, and over the keys of the two last buckets
  float x[MAPS], m[MAPS], xl[MAPS], xr[MAPS], ml[MAPS], mr[MAPS], far_l = 0.f, far_r = 0.f;
#pragma unroll
  for (int a = 0; a < MAPS; ++a) x[a] = m[a] = xl[a] = xr[a] = ml[a] = mr[a] = 0.f;
  // 32 NT keys from position key0 on, their fragments from ka and va
  const auto work = [&](const auto& ka, const auto& va, int key0, auto wide_rows) __attribute__((always_inline)) {
    constexpr bool WIDE_HEAD = decltype(wide_rows)::value;
    const int klast = key0 + 32 * NT - 1;
    if (p.causal && key0 > qhi) return;
    const bool whole = klast < kend && (!p.causal || klast <= qlo);
    const float* tb = tab + (reach + PAD) + key0 - qpos + 4 * half;
    float far = 0.f;
    int side = 0;
    bool near = false;
    if (p.bk.n) {
      if (klast - qlo <= -reach) far = tab[PAD], side = -1;
      else if (key0 - qhi >= reach) far = tab[2 * (reach + PAD)], side = 1;
      else near = true;
      if (WIDE_HEAD) far = 4.f * (far - base);
    }
    f32x16 da[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      da[t] = zero16();
#pragma unroll
      for (int i = 0; i < D / 16; ++i) da[t] = mma(va.frag(32 * t, i), gf[i], da[t]);
    }
#pragma unroll
    for (int a = 0; a < MAPS; ++a) {
      f32x16 s[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        s[t] = zero16();
#pragma unroll
        for (int i = 0; i < W / 16; ++i) s[t] = mma(ka.frag(32 * t, a * (W / 16) + i), qf[a * (W / 16) + i], s[t]);
      }
      float cc = c, off = far - lse[a];
      if (near || !whole) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int k = 32 * t + 8 * (r >> 2) + (r & 3);
            if (WIDE_HEAD && r % 4 == 0) few_at_a_time();
            s[t][r] = fmaf(s[t][r], c, near ? (WIDE_HEAD ? 4.f * (tb[k] - base) : tb[k]) : far);
          }
        if (!whole) {
          const int last = min(kend - 1, p.causal ? qpos : 0x7fffffff) - key0 - 4 * half;     // last visible key
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (32 * t + 8 * (r >> 2) + (r & 3) > last) s[t][r] = -INFINITY;
        }
        cc = 1.f;
        off = -lse[a];
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] = exp2_(fmaf(s[t][r], cc, off));
      if (sums) {
        float xs = 0.f, ms = 0.f;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            xs = fmaf(s[t][r], da[t][r], xs);
            ms += s[t][r];
          }
        x[a] += xs, m[a] += ms;
        if (side < 0) xl[a] += xs, ml[a] += ms;
        if (side > 0) xr[a] += xs, mr[a] += ms;
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] *= (a == 0 ? da[t][r] : -lam * da[t][r]) - delta[a];
      if (p.part && !side) {
        // [distance key - query + 31][query]: a lane writes its query's column, then lane l sums row l (63 of them); what lies
        // outside the 32 x 32 tile stays zero from the start
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float* at = scr + (31 - (lane & 31) + 4 * half) * SCR + (lane & 31);
#pragma unroll
          for (int r = 0; r < 16; ++r) at[(8 * (r >> 2) + (r & 3)) * SCR] = s[t][r];
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = 0; q < 8; ++q) sum += *(const f32x4*)(scr + lane * SCR + 4 * q);
          if (lane < 63) diag[(reach + PAD) + key0 + 32 * t - qlo + lane - 31] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          Frag<T> sf;
          to_frag(sf, s[t], 8 * u);
#pragma unroll
          for (int j = 0; j < W / 32; ++j)
            acc[a * (W / 32) + j] = mma(ka.frag_t(32 * t + 16 * u, a * W + 32 * j), sf, acc[a * (W / 32) + j]);
        }
    }
  };
  const auto walk = [&](auto wide_rows) __attribute__((always_inline)) {
    if constexpr (SPLIT) {
      for (int k0 = 32 * wave; k0 < kend; k0 += 128) work(InMemory{kb, p.ks, k0, kend, lane}, InMemory{vb, p.vs, k0, kend, lane}, k0, wide_rows);
    } else {
      Stream<T, D> kv(lds);
      if (kend > 0) kv.next(kb, p.ks, vb, p.vs, 0, kend, tid);
      for (int k0 = 0; k0 < kend; k0 += TK::ROWS) {
        kv.arrive();
        if (k0 + TK::ROWS < kend) kv.next(kb, p.ks, vb, p.vs, k0 + TK::ROWS, kend, tid);
#pragma unroll 1
        for (int t0 = 0; t0 < TK::ROWS / 32; t0 += NT)
          if (k0 + 32 * t0 < kend) work(Staged<T, D>{kv.a(), 32 * t0, lane}, Staged<T, D>{kv.b(), 32 * t0, lane}, k0 + 32 * t0, wide_rows);
      }
    }
  };
  if (wide) walk(std::true_type{});        // a loop of its own: in one loop with the ordinary tiles it cost those 3 to 5 %
  else walk(std::false_type{});
  if (min(kend - 1, p.causal ? qpos : 0x7fffffff) < 0)               // a query that sees no key takes no gradient, whatever keys and values hold
#pragma unroll
    for (int j = 0; j < D / 32; ++j) acc[j] = zero16();
  if constexpr (SPLIT) {
    // the waves' sums over their keys: statistics into every wave, the output tile through the same LDS
    float* st = (float*)lds;
#pragma unroll
    for (int a = 0; a < MAPS; ++a) {
      float* v[6] = {&x[a], &m[a], &xl[a], &xr[a], &ml[a], &mr[a]};
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 6; ++i) st[(wave * 6 + i) * 64 + lane] = *v[i];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 6; ++i) *v[i] = (st[i * 64 + lane] + st[(6 + i) * 64 + lane]) + (st[(12 + i) * 64 + lane] + st[(18 + i) * 64 + lane]);
    }
  }
#pragma unroll
  for (int a = 0; a < MAPS; ++a) {
    x[a] = column_sum(x[a]);
    m[a] = column_sum(m[a]);
    x[a] = m[a] == 0.f ? 0.f : x[a] / m[a];     // a NaN stays one
    const float w = a == 0 ? 1.f : -lam;
    if (sums && live && half == 0 && (!SPLIT || wave == 0)) p.delta[(((size_t)b * p.H + h) * MAPS + a) * p.Sq + qrow] = w * x[a];
    far_l += w * (xl[a] - x[a] * ml[a]);        // both halves: the sum over the wave adds their keys
    far_r += w * (xr[a] - x[a] * mr[a]);
  }
  if constexpr (SPLIT) {
    if (wave) far_l = far_r = 0.f;                               // the statistics are the same in every wave
    meet_sum<T, D>((float*)lds, acc, p.scale, (T*)p.dq + ((size_t)b * p.Sq * p.H + h) * D, (long long)p.H * D, row0, p.Sq, wave, lane);
  } else if (live) {
    T* dq = (T*)p.dq + orow;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        store4(dq + 32 * j + 8 * g + 4 * half, p.scale * acc[j][4 * g], p.scale * acc[j][4 * g + 1], p.scale * acc[j][4 * g + 2],
               p.scale * acc[j][4 * g + 3]);
  }
  // partial sums of this block: bucket sums of the four waves' distances, lambda
  const size_t slot = ((size_t)h * p.B + b) * tiles + tile;
  if (p.part) {
    __syncthreads();
    float* fars = (float*)lds;                                     // the tiles are done
    far_l = wave_sum(far_l);
    far_r = wave_sum(far_r);
    if (lane == 0) {
      fars[2 * wave] = far_l;
      fars[2 * wave + 1] = far_r;
    }
    // the four waves' sums into the first
    float* d0 = tab + ntab;
    for (int i = tid; i < ntab; i += 256) {
      float sum = d0[i];
      for (int w = 1; w < 4; ++w) sum += d0[w * ntab + i];
      d0[i] = sum;
    }
    __syncthreads();
    const float* mid = d0 + reach + PAD;
    for (int u = tid; u < p.bk.n; u += 256) {
      const int right = p.bk.two_sided && u >= p.bk.side, i = right ? u - p.bk.side : u, last = p.bk.side - 1;
      const int a = first_distance(p.bk, i), z = i == last ? reach + PAD + 1 : first_distance(p.bk, i + 1);    // distances a .. z - 1; behind them the far sums
      float sum = 0.f;
#pragma unroll 8
      for (int n = a; n < z; ++n) sum += right ? (n > 0 ? mid[n] : 0.f) : mid[-n];
      if (i == last)
        for (int w = 0; w < 4; ++w) sum += fars[2 * w + right];
      if (!p.bk.two_sided && i == 0) {                                     // one-sided: everything ahead is distance 0
#pragma unroll 8
        for (int n = 1; n <= reach + PAD; ++n) sum += mid[n];
        for (int w = 0; w < 4; ++w) sum += fars[2 * w + 1];
      }
      p.part[slot * p.bk.n + u] = sum;
    }
  }
  if constexpr (MAPS == 2) {
    if (p.lam_part) {
      const float xs = wave_sum(half == 0 && (!SPLIT || wave == 0) ? x[1] : 0.f);
      __shared__ float lams[4];
      if (lane == 0) lams[wave] = xs;
      __syncthreads();
      if (tid == 0) p.lam_part[slot] = -(lams[0] + lams[1] + lams[2] + lams[3]);
    }
  }
}

template <typename T, int D, int MAPS> constexpr bool v_in_lds() { return sizeof(T) == 2 && D == 128 && MAPS == 1; }
template <typename T, int D, int MAPS> constexpr int dkv_head() {
  return v_in_lds<T, D, MAPS>() ? Stream<T, D, 32>::BYTES + Tile<T, D, 128>::BYTES : Stream<T, D>::BYTES;
}

// floats that dK/dV holds for a tile's rows
template <int MAPS> constexpr int row_floats() { return (4 * MAPS + 1) * TILE; }

template <typename T, int D, int MAPS, bool SPLIT>
__global__ __launch_bounds__(256, D == 32 && !SPLIT ? 3 : sizeof(T) == 2 && D * MAPS <= 128 ? 2 : 1) void attn_dkv_kernel(const Params p) {
  // bf16 at 128 columns, one map: two waves per SIMD leave 256 registers each, 160 of them accumulators and keys; the block's values stay in
  // LDS, and the stream's tiles are half as long, so that two blocks share a CU
  constexpr bool VLDS = v_in_lds<T, D, MAPS>();
  using TK = Tile<T, D, VLDS ? 32 : tile_rows<T, D>()>;
  using VT = Tile<T, D, 128>;
  constexpr int W = D / MAPS;
  constexpr int NT = sizeof(T) == 2 && D * MAPS <= 64 ? 2 : 1, KB = SPLIT ? 32 : 128, STEP = SPLIT ? 32 : TK::ROWS;     // 32-query tiles worked on together, as the registers allow
  extern __shared__ __attribute__((aligned(16))) char lds[];
  // [MAPS][4][TILE]: delta, and -lse alone and with the bias of either last bucket (all a plain tile needs of it), then the rows'
  // bases; one set in use while the next is written, or one for each wave
  constexpr int ROWS = row_floats<MAPS>();
  float* rows2 = (float*)(lds + (SPLIT ? meet_bytes<D>() : (int)dkv_head<T, D, MAPS>()));
  float* tab0 = rows2 + (SPLIT ? 4 : 2) * ROWS;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int n = p.B * p.Hkv, G = p.H / p.Hkv, reach = p.bk.reach;
  float* tab = tab0 + (SPLIT && p.bk.n ? wave * (2 * (reach + PAD) + 1) : 0);
  const int share = (int)blockIdx.x % p.parts, block = (int)blockIdx.x / p.parts, j0 = block % n, kblock = block / n * KB, b = j0 / p.Hkv, hk = j0 % p.Hkv;
  const int start = uniform(start_of(p, b));
  int limit = uniform(key_limit(p, b));
  if (p.causal) limit = max(0, min(limit, start + p.Sq));         // keys behind the last query: seen by none, not read, no gradient
  const int klo = kblock + (SPLIT ? 0 : 32 * wave), krow = klo + (lane & 31), khi = klo + 31;
  const bool live = krow < limit;
  const T* kp = (const T*)p.k + b * p.kb + hk * p.kh + (long long)krow * p.ks;
  const T* vp = (const T*)p.v + b * p.vb + hk * p.vh + (long long)krow * p.vs;
  // fp32 at 128 columns: keys, values and both accumulators do not fit in 512 registers; the values come from the cache again for
  // every tile (16 KiB against 8192 cycles of matrix instructions)
  constexpr bool HOLD = sizeof(T) * D <= 256 && !VLDS;
  Frag<T> kf[D / 16], vf[HOLD ? D / 16 : 1];
  f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    kf[i] = frag_global(kp, i, lane, live);
    if constexpr (HOLD) vf[i] = frag_global(vp, i, lane, live);
  }
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    dk[j] = zero16();
    dv[j] = zero16();
  }
  const float c = positive_scale(p.scale, kf);
  int first = 0;                                                  // first query row that sees a key of this block
  if (p.causal) first = max(0, kblock - start) / STEP * STEP;
  const int per = kblock < limit && first < p.Sq ? (p.Sq - first + STEP - 1) / STEP : 0, total = per * G;
  float rl[MAPS], rd[MAPS], lam = 0.f, far_l = 0.f, far_r = 0.f;
  // lse and delta of STEP rows from q0 on, one row per thread of `t`
  const auto fetch_rows = [&](int h, int q0, int t) {
    if (t < STEP)
#pragma unroll
      for (int a = 0; a < MAPS; ++a) {
        const size_t at = (((size_t)b * p.H + h) * MAPS + a) * p.Sq + q0 + t;
        rl[a] = q0 + t < p.Sq ? p.lse[at] : INFINITY;
        rd[a] = q0 + t < p.Sq ? p.delta[at] : 0.f;
      }
  };
  const auto put_rows = [&](float* rows, int h, int q0, int t, auto wide_heads) {
    if (t < STEP) {
      float l = far_l, r = far_r;
      if constexpr (decltype(wide_heads)::value) {
        float base = 0.f;
        if (p.wide[h]) base = q0 + t < p.Sq ? p.base[((size_t)b * p.H + h) * p.Sq + q0 + t] : 3.4e38f;         // behind the last row: above any entry
        rows[MAPS * 4 * TILE + t] = base;
        l = 4.f * (l - base);
        r = 4.f * (r - base);
      }
#pragma unroll
      for (int a = 0; a < MAPS; ++a) {
        float* at = rows + a * 4 * TILE + t;
        at[0] = rd[a];
        at[TILE] = -rl[a];
        at[2 * TILE] = l - rl[a];
        at[3 * TILE] = r - rl[a];
        if constexpr (decltype(wide_heads)::value)
          if (rl[a] == INFINITY) at[2 * TILE] = at[3 * TILE] = -INFINITY;
      }
    }
  };
  char* vlds = lds + Stream<T, D, TK::ROWS>::BYTES;
  const auto v_frag = [&](int i) __attribute__((always_inline)) {
    if constexpr (HOLD) return vf[i];
    else if constexpr (VLDS) return VT::frag(vlds, 32 * wave, i, lane);
    else return frag_global(vp, i, lane, live);
  };
  // 32 NT queries from row r0 on, their fragments from qa and ga, their offsets at `rows`
  const auto work = [&](const auto& qa, const auto& ga, const float* rows, int r0, auto wide_heads) __attribute__((always_inline)) {
    constexpr bool WIDE_HEADS = decltype(wide_heads)::value;
    const int qlo = start + r0, qhi = qlo + 32 * NT - 1;
    if (r0 >= p.Sq || klo >= limit || (p.causal && qhi < klo)) return;
    const bool whole = khi < limit && (!p.causal || khi <= qlo);
    const float* tb = tab + (reach + PAD) + krow - qlo - 4 * half;
    int offs = TILE;                                                 // which of a row's offsets
    bool near = false;
    if (p.bk.n) {
      if (khi - qlo <= -reach) offs = 2 * TILE;
      else if (klo - qhi >= reach) offs = 3 * TILE;
      else near = true;
    }
    // one wave per SIMD: the second products' operands are requested before the scores' long way through exp2 (4 x 8 x 2048 causal,
    // training as a whole: 377 -> 358 us)
    constexpr bool EARLY = sizeof(T) == 2 && D == 128 && MAPS == 2;
    Frag<T> qt[EARLY ? 2 * D / 32 : 1], gt[EARLY ? 2 * D / 32 : 1];
    f32x16 da[NT], mix[MAPS == 2 ? NT : 1];
    const auto add_dv = [&](const f32x16 (&w)[NT]) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          Frag<T> pf;
          to_frag(pf, w[t], 8 * u);
#pragma unroll
          for (int j = 0; j < D / 32; ++j) dv[j] = mma(EARLY ? gt[EARLY ? u * (D / 32) + j : 0] : ga.frag_t(32 * t + 16 * u, 32 * j), pf, dv[j]);
        }
    };
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      da[t] = zero16();
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        da[t] = mma(ga.frag(32 * t, i), v_frag(i), da[t]);
    }
#pragma unroll
    for (int a = 0; a < MAPS; ++a) {
      f32x16 s[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        s[t] = zero16();
#pragma unroll
        for (int i = 0; i < W / 16; ++i) s[t] = mma(qa.frag(32 * t, a * (W / 16) + i), kf[a * (W / 16) + i], s[t]);
      }
      if constexpr (EARLY) {
        if (a == 0)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
              qt[u * (D / 32) + j] = qa.frag_t(16 * u, 32 * j);
              gt[u * (D / 32) + j] = ga.frag_t(16 * u, 32 * j);
            }
      }
      const float* ls = rows + a * 4 * TILE + 4 * half;
      float cc = c;
      if (near) {
        const float* bs = rows + MAPS * 4 * TILE + 4 * half;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int q = 32 * t + 8 * (r >> 2) + (r & 3);
            if (WIDE_HEADS && r % 4 == 0) few_at_a_time();
            s[t][r] = fmaf(s[t][r], c, WIDE_HEADS ? 4.f * (tb[-q] - bs[q]) : tb[-q]);
          }
        cc = 1.f;
      }
      if (!whole) {       // first query that sees this key
        const int first = krow >= limit ? 0x7fffffff : (p.causal ? krow - qlo - 4 * half : -0x7fffffff);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (32 * t + 8 * (r >> 2) + (r & 3) < first) s[t][r] = -INFINITY;
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 nl = *(const f32x4*)(ls + offs + 32 * t + 8 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t][4 * g + e] = exp2_(fmaf(s[t][4 * g + e], cc, nl[e]));
        }
      if constexpr (MAPS == 2) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) mix[t][r] = a == 0 ? s[t][r] : fmaf(-lam, s[t][r], mix[t][r]);
        if (a == 1) add_dv(mix);
      } else {
        add_dv(s);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 dl = *(const f32x4*)(ls + 32 * t + 8 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t][4 * g + e] *= (a == 0 ? da[t][4 * g + e] : -lam * da[t][4 * g + e]) - dl[e];
        }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          Frag<T> sf;
          to_frag(sf, s[t], 8 * u);
#pragma unroll
          for (int j = 0; j < W / 32; ++j)
            dk[a * (W / 32) + j] = mma(EARLY ? qt[EARLY ? u * (D / 32) + a * (W / 32) + j : 0] : qa.frag_t(32 * t + 16 * u, a * W + 32 * j), sf, dk[a * (W / 32) + j]);
        }
    }
  };
  const T* q_of = (const T*)p.q + b * p.qb;
  const T* g_of = (const T*)p.d_o + (size_t)b * p.Sq * p.H * D;
  const auto walk = [&](auto wide_heads, int tid, int lane) __attribute__((always_inline)) {
    asm volatile("" : "+v"(tid), "+v"(lane));   // nothing in common with the other kind's walk: what both would share costs the registers
    if constexpr (SPLIT) {                      // that the products' operands are requested into (16 x 8 x 1024 x 64: 108 us, else 117)
      float* rows = rows2 + wave * ROWS;
      int held = -1;
      for (int it = wave; it < total; it += 4) {
        const int h = hk * G + it / per, q0 = first + it % per * STEP;
        fetch_rows(h, q0, lane);
        if (h != held) {
          held = h;
          if constexpr (MAPS == 2) lam = ldf(p.lam, h, p.lam_f32);
          if (p.bk.n) {
            fill_bias(p, tab, h, lane, 64, wide_heads);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            far_l = tab[PAD];
            far_r = tab[2 * (reach + PAD)];
          }
        }
        put_rows(rows, h, q0, lane, wide_heads);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        work(InMemory{q_of + h * p.qh, p.qs, q0, p.Sq, lane}, InMemory{g_of + (size_t)h * D, (long long)p.H * D, q0, p.Sq, lane}, rows, q0, wide_heads);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
    } else {
      Stream<T, D, TK::ROWS> qg(lds);
      const auto fetch = [&](int it) {
        const int h = hk * G + it / per, q0 = first + it % per * STEP;
        qg.next(q_of + h * p.qh, p.qs, g_of + (size_t)h * D, (long long)p.H * D, q0, p.Sq, tid);
        fetch_rows(h, q0, tid);
      };
      // this block's part of the (head, query tile) list
      const int it0 = (int)((long long)total * share / p.parts), it1 = (int)((long long)total * (share + 1) / p.parts);
      if (VLDS && it0 < it1) VT::dma((const T*)p.v + b * p.vb + hk * p.vh, p.vs, kblock, limit, vlds, tid);
      if (it0 < it1) fetch(it0);
      for (int it = it0; it < it1; ++it) {
        const int h = hk * G + it / per, q0 = first + it % per * STEP;
        float* rows = rows2 + (it & 1) * ROWS;          // written while other waves may still read the other one
        if (it == it0 || it % per == 0) {                             // a head begins
          if constexpr (MAPS == 2) lam = ldf(p.lam, h, p.lam_f32);
          if (p.bk.n) {
            __syncthreads();
            fill_bias(p, tab, h, tid, 256, wide_heads);
            __syncthreads();
            far_l = tab[PAD];
            far_r = tab[2 * (reach + PAD)];
          }
        }
        put_rows(rows, h, q0, tid, wide_heads);
        qg.arrive();
        if (it + 1 < it1) fetch(it + 1);
#pragma unroll 1
        for (int t0 = 0; t0 < TK::ROWS / 32; t0 += NT)
          work(Staged<T, D, TK::ROWS>{qg.a(), 32 * t0, lane}, Staged<T, D, TK::ROWS>{qg.b(), 32 * t0, lane}, rows + 32 * t0, q0 + 32 * t0, wide_heads);
      }
    }
  };
  bool wide = false;                                               // one of the key head's heads is
  if (p.bk.n) {
    for (int g = lane; g < G; g += 64) wide = wide || p.wide[hk * G + g];
    wide = __any(wide);
  }
  if (wide) walk(std::true_type{}, tid, lane);
  else walk(std::false_type{}, tid, lane);
  int end = limit;
  asm volatile("" : "+s"(end));                                     // compared anew, for the same reason as above
  if (krow >= end)                                                  // keys that no query sees take no gradient, not even of a NaN in dO or Q
#pragma unroll
    for (int j = 0; j < D / 32; ++j) dk[j] = dv[j] = zero16();
  if constexpr (SPLIT) {
    const long long ld = (long long)p.Hkv * D;
    meet_sum<T, D>((float*)lds, dk, p.scale, (T*)p.dk + ((size_t)b * p.Sk * p.Hkv + hk) * D, ld, klo, p.Sk, wave, lane);
    meet_sum<T, D>((float*)lds, dv, 1.f, (T*)p.dv + ((size_t)b * p.Sk * p.Hkv + hk) * D, ld, klo, p.Sk, wave, lane);
    return;
  }
  if (krow < p.Sk) {
    const size_t at = (((size_t)b * p.Sk + krow) * p.Hkv + hk) * D;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * j + 8 * g + 4 * half;
        if (p.parts > 1) {
          const size_t pt = (size_t)share * p.B * p.Sk * p.Hkv * D + at + d;
          store4(p.dk_part + pt, p.scale * dk[j][4 * g], p.scale * dk[j][4 * g + 1], p.scale * dk[j][4 * g + 2], p.scale * dk[j][4 * g + 3]);
          store4(p.dv_part + pt, dv[j][4 * g], dv[j][4 * g + 1], dv[j][4 * g + 2], dv[j][4 * g + 3]);
          continue;
        }
        store4((T*)p.dk + at + d, p.scale * dk[j][4 * g], p.scale * dk[j][4 * g + 1], p.scale * dk[j][4 * g + 2], p.scale * dk[j][4 * g + 3]);
        store4((T*)p.dv + at + d, dv[j][4 * g], dv[j][4 * g + 1], dv[j][4 * g + 2], dv[j][4 * g + 3]);
      }
  }
}

// dk and dv from their parts, four values per thread, in the parts' order
template <typename T> __global__ __launch_bounds__(256) void attn_parts_kernel(const Params p, long long n) {
  const long long i = 4 * ((long long)blockIdx.x * 256 + threadIdx.x);
  if (i >= n) return;
  f32x4 a = *(const f32x4*)(p.dk_part + i), b = *(const f32x4*)(p.dv_part + i);
  for (int k = 1; k < p.parts; ++k) {
    a += *(const f32x4*)(p.dk_part + k * n + i);
    b += *(const f32x4*)(p.dv_part + k * n + i);
  }
  store4((T*)p.dk + i, a[0], a[1], a[2], a[3]);
  store4((T*)p.dv + i, b[0], b[1], b[2], b[3]);
}

// table gradient [n][H] and lambda gradient [H] from the blocks' partial sums; one wave per value, fp64, fixed order
__global__ __launch_bounds__(64) void attn_fold_kernel(const float* part, const float* lam_part, void* dbias, void* dlam, int n, int H,
                                                       int slots, int bias_f32, int lam_f32) {
  const int h = (int)blockIdx.x % H, u = (int)blockIdx.x / H, lane = threadIdx.x;
  const bool lam = u == n;
  double sum = 0.0;
  for (int s = lane; s < slots; s += 64) {
    const size_t at = (size_t)h * slots + s;
    sum += lam ? lam_part[at] : part[at * n + u];
  }
  sum = wave_sum_d(sum);
  if (lane) return;
  void* out = lam ? dlam : dbias;
  const size_t at = lam ? (size_t)h : (size_t)u * H + h;
  if (lam ? lam_f32 : bias_f32) ((float*)out)[at] = (float)sum;
  else ((__bf16*)out)[at] = (__bf16)(float)sum;
}

struct Sizes {
  size_t delta, base, wide, part, lam, dkv;      // floats; dkv: of each of dk's and dv's parts together
  int slots, parts;
  size_t floats() const { return delta + base + wide + part + lam + 2 * dkv; }
};
constexpr int CUS = 256;
bool split_rows(const eovae_token_attention* d) {
  return d->dtype == EOVAE_F32 && (long long)d->batch * d->heads * ((d->sq + 127) / 128) < CUS;
}
bool split_keys(const eovae_token_attention* d) {
  return d->dtype == EOVAE_F32 && (long long)d->batch * d->kv_heads * ((d->sk + 127) / 128) < CUS;
}
Sizes sizes_of(const Params& p, const eovae_token_attention* d, bool dbias, bool dlam) {
  Sizes s;
  const int maps = d->maps, rb = split_rows(d) ? 32 : 128;
  s.slots = p.B * ((p.Sq + rb - 1) / rb);
  s.delta = ((size_t)p.B * p.H * maps * p.Sq + 3) & ~(size_t)3;
  s.base = p.bk.n ? ((size_t)p.B * p.H * p.Sq + 3) & ~(size_t)3 : 0;
  s.wide = p.bk.n ? ((size_t)p.H + 3) & ~(size_t)3 : 0;
  s.part = dbias ? ((size_t)s.slots * p.H * p.bk.n + 3) & ~(size_t)3 : 0;
  s.lam = dlam ? ((size_t)s.slots * p.H + 3) & ~(size_t)3 : 0;
  // Few key heads and a long key axis leave CUs without a block (and, causal, one long row of blocks): the queries are cut into
  // parts until there are two blocks per CU, and dk, dv are joined from fp32 parts.
  const long long blocks = (long long)d->batch * d->kv_heads * ((d->sk + 127) / 128), items = (long long)(d->heads / d->kv_heads) * ((d->sq + 127) / 128);
  long long parts = split_keys(d) || blocks > CUS ? 1 : 2 * CUS / blocks;
  if (parts > 8) parts = 8;
  if (parts > items) parts = items;
  s.parts = (int)parts;
  s.dkv = parts > 1 ? (size_t)parts * p.B * p.Sk * p.Hkv * d->dim : 0;
  return s;
}

template <typename T, int D, int MAPS> int run_bwd(Params& p, const eovae_token_attention* d, hipStream_t st) {
  const char* who = "token_attention_bwd";
  const Sizes s = sizes_of(p, d, d->dbias, d->dlam);
  const size_t need = 4 * s.floats();
  EOVAE_CHECK_ARG(d->ws && d->ws_bytes >= need, "%s: workspace of %zu bytes, needs %zu", who, d->ws_bytes, need);
  p.delta = (float*)d->ws;
  p.base = p.delta + s.delta;
  p.wide = (int*)(p.base + s.base);
  float* rest = p.base + s.base + s.wide;
  if (d->dbias) p.part = rest;
  if (d->dlam) p.lam_part = rest + s.part;
  p.parts = s.parts;
  if (s.parts > 1) {
    p.dk_part = rest + s.part + s.lam;
    p.dv_part = p.dk_part + s.dkv;
  }
  const size_t tiles = (size_t)Stream<T, D>::BYTES, tab = 4 * (size_t)bias_entries(p.bk);
  const size_t sums = d->dbias ? 4 * tab + 16 + 4 * 4 * SCR_FLOATS : 0;
  const size_t rows = 4 * row_floats<MAPS>();
  int rc = EOVAE_OK;
  const auto dq = [&](auto kernel, int rb, size_t head) {
    return launch(kernel, (size_t)((p.Sq + rb - 1) / rb) * p.B * p.H, 256, head + tab + sums, p, st, who);
  };
  const auto dkv = [&](auto kernel, int kb, size_t head, int copies) {
    return launch(kernel, (size_t)((p.Sk + kb - 1) / kb) * p.B * p.Hkv * p.parts, 256, head + copies * rows + (copies == 4 ? 4 : 1) * tab, p, st, who);
  };
  if constexpr (sizeof(T) == 4) {
    const size_t meet = meet_bytes<D>();
    rc = split_rows(d) ? dq(attn_dq_kernel<T, D, MAPS, true>, 32, meet) : dq(attn_dq_kernel<T, D, MAPS, false>, 128, tiles);
    if (rc == EOVAE_OK) rc = split_keys(d) ? dkv(attn_dkv_kernel<T, D, MAPS, true>, 32, meet, 4) : dkv(attn_dkv_kernel<T, D, MAPS, false>, 128, dkv_head<T, D, MAPS>(), 2);
  } else {
    rc = dq(attn_dq_kernel<T, D, MAPS, false>, 128, tiles);
    if (rc == EOVAE_OK) rc = dkv(attn_dkv_kernel<T, D, MAPS, false>, 128, dkv_head<T, D, MAPS>(), 2);
  }
  if (rc) return rc;
  if (p.parts > 1) {
    const long long n = (long long)p.B * p.Sk * p.Hkv * D;
    EOVAE_CHECK_ARG((n + 1023) / 1024 <= 0x7fffffff, "%s: %lld values of dk", who, n);
    hipLaunchKernelGGL(attn_parts_kernel<T>, dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, st, p, n);
    EOVAE_CHECK_LAUNCH(who);
  }
  const int nb = d->dbias ? p.bk.n : 0, outs = nb + (d->dlam ? 1 : 0);
  if (outs == 0) return EOVAE_OK;
  hipLaunchKernelGGL(attn_fold_kernel, dim3((unsigned)(p.H * outs)), dim3(64), 0, st, p.part, p.lam_part, d->dbias, d->dlam, nb, p.H, s.slots,
                     p.bias_f32, p.lam_f32);
  EOVAE_CHECK_LAUNCH(who);
  return EOVAE_OK;
}

}  // namespace

size_t tok_fwd_workspace(const eovae_token_attention* d, const Params& p);

extern "C" {
size_t eovae_token_attention_workspace(const eovae_token_attention* d, int backward) {
  Params p;
  if (make_params(d, p, "token_attention_workspace", 0)) return 0;
  if (!backward) return tok_fwd_workspace(d, p);
  const Sizes s = sizes_of(p, d, d->bias != nullptr, d->maps == 2);
  return 4 * s.floats();
}
int eovae_token_attention_bwd(const eovae_token_attention* d, void* stream) {
  Params p;
  const int rc = make_params(d, p, "token_attention_bwd", 1);
  if (rc) return rc;
  return TOK_DISPATCH(d, run_bwd, p, d, (hipStream_t)stream);
}
}
