// Fused attention forward with bucketed relative position bias, one or two softmax maps (token_attn_common.h).
//
// Row form: a block owns 128 (two maps: 64) query rows of one head and walks the keys once, 64 at a time, with the running
// maximum and sum of every row's softmax; a lane owns ONE query (its column of S^T = K Q^T), so the statistics are plain
// registers and the other half of a column is one cross-lane exchange away.  Two maps: waves 0, 1 hold map 0, waves 2, 3
// map 1 of the same rows (same K / V tiles, half of K's columns each) and meet once at the end.  One wave reads 32 KiB of LDS
// for 1024 cycles of matrix instructions at 128 columns, which is what the four waves' share of the LDS gives, and 32 exp2 at a
// quarter of the vector rate beside them; two waves per SIMD overlap the three.  Measured: 16 heads x 8191 causal x 128
// columns 301 us (910 TFLOP/s), 16 x 8 x 1024 x 64 57 us without a bias (600), two maps 16 x 8 x 1000 ragged 105 .. 126 us.
// Step form (few rows per key head, e.g. single tokens against a cache, or a call too small to fill the chip): the rows are the
// query heads that share one key head times the query tokens, 32 of them to a block, the four waves take different keys, the
// key axis is also split over blocks where it is long, and then a second kernel joins the partial sums.  Bound by bytes where a
// cache is long: 32 caches of 1024 .. 4096 keys x 4 key heads x 128, bf16, 42 us (4.0 TB/s; copies reach 4.9) and 4 for the join.
#include <math.h>
#include <type_traits>
#include "token_attn_common.h"

using namespace tok;

namespace {

constexpr int CUS = 256;
constexpr int SPLIT_KEYS = 512;        // fewest keys of a split where a call has more than 32 rows per key head

// Scores of one wave's 32 queries against 32 NT keys, turned into probabilities in place (relative to 2^m, not normalised);
// returns the factor by which the wave's earlier sums have to be multiplied (`moved`: whether any lane's differs from 1).
// The reference m of a row is its maximum when it last moved: it follows only when a score passes it by 2^SLACK, which the
// fp32 sums hold easily and which saves rescaling the output tile for almost every key tile.
// Plain tiles (all pairs visible, one bias value) cost one fma and one exp2 per score; the others add bias and mask first.
constexpr float SLACK = 8.f;
template <int NT, bool WIDE_HEAD>
__device__ __forceinline__ float softmax_tile(const Params& p, f32x16 (&s)[NT], float& m, float& l, bool& moved, float c, int key0, int limit,
                                              int qpos, int qlo, int qhi, const float* tab, float base, int lane) {
  const int half = lane >> 5, klast = key0 + 32 * NT - 1;
  const bool whole = klast < limit && (!p.causal || klast <= qlo);
  float far = 0.f;
  bool near = false;
  if (p.bk.n) {
    const int reach = p.bk.reach;
    if (klast - qlo <= -reach) far = tab[PAD];                              // every pair at or behind the last border
    else if (key0 - qhi >= reach) far = tab[2 * (reach + PAD)];
    else near = true;
    if (WIDE_HEAD) far = 4.f * (far - base);
  }
  if (near || !whole) {
    const float* tb = tab + (p.bk.reach + PAD) + key0 - qpos + 4 * half;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int k = 32 * t + 8 * (r >> 2) + (r & 3);
        if (WIDE_HEAD && r % 4 == 0) few_at_a_time();
        s[t][r] = fmaf(s[t][r], c, near ? (WIDE_HEAD ? 4.f * (tb[k] - base) : tb[k]) : far);
      }
    if (!whole) {
      // last visible key of this lane's query, relative to its first score
      const int last = min(limit - 1, p.causal ? qpos : 0x7fffffff) - key0 - 4 * half;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * t + 8 * (r >> 2) + (r & 3) > last) s[t][r] = -INFINITY;
    }
    c = 1.f;
    far = 0.f;
  }
  float top = s[0][0];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[t][r]);
  top = fmaf(column_max(top), c, far);
  float a = 1.f;
  moved = __any(top > m + SLACK);
  if (moved) {
    const float mn = fmaxf(m, top);
    a = exp2_(m - (mn == -INFINITY ? 0.f : mn));                             // m = -inf: 0
    m = mn;
    l *= a;
  }
  const float off = far - (m == -INFINITY ? 0.f : m);
  float sum = 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[t][r] = exp2_(fmaf(s[t][r], c, off));
      sum += s[t][r];
    }
  l += sum;
  return a;
}

// One wave's pass over a staged tile of TILE keys: scores of its 32 queries, softmax update, O^T += V^T P^T.
// Probabilities enter the value product in the tensors' type (to_frag): bf16 rounds each once.
// r0: first row of the tile in LDS, key0: its position; qpos: this lane's query position; limit: keys visible at all.
template <typename T, int D, int MAPS> constexpr int row_tile() { return sizeof(T) == 2 && D == 128 && MAPS == 2 ? 32 : tile_rows<T, D>(); }
template <typename T, int D, int R, int W, int NT, bool WIDE_HEAD>
__device__ __forceinline__ void tile_step(const Params& p, char* lk, char* lv, const Frag<T> (&qf)[W / 16], f32x16 (&acc)[D / 32],
                                          float& m, float& l, float c, int map, int r0, int key0, int limit, int qpos, int qlo, int qhi, const float* tab,
                                          float base, int lane) {
  using TK = Tile<T, D, R>;
  f32x16 s[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    s[t] = zero16();
#pragma unroll
    for (int i = 0; i < W / 16; ++i) s[t] = mma(TK::frag(lk, r0 + 32 * t, map * (W / 16) + i, lane), qf[i], s[t]);
  }
  bool moved;
  const float a = softmax_tile<NT, WIDE_HEAD>(p, s, m, l, moved, c, key0, limit, qpos, qlo, qhi, tab, base, lane);
  if (moved)
#pragma unroll
    for (int j = 0; j < D / 32; ++j) acc[j] *= a;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      Frag<T> pf;
      to_frag(pf, s[t], 8 * u);
#pragma unroll
      for (int j = 0; j < D / 32; ++j) acc[j] = mma(TK::frag_t(lv, r0 + 32 * t + 16 * u, 32 * j, lane), pf, acc[j]);
    }
}

template <typename T, int D, int MAPS>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? (D <= 64 ? 4 : MAPS == 2 ? 3 : 2) : D == 32 ? 3 : 1) void attn_rows_kernel(const Params p) {
  constexpr int W = D / MAPS;                 // width of one map's queries and keys
  constexpr int RB = 128 / MAPS;              // query rows of a block
  extern __shared__ __attribute__((aligned(16))) char lds[];
  float* tab = (float*)(lds + Stream<T, D, row_tile<T, D, MAPS>()>::BYTES);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int map = MAPS == 2 ? wave >> 1 : 0, wrow = 32 * (MAPS == 2 ? (wave & 1) : wave);
  const int nbh = p.B * p.H, tiles = (p.Sq + RB - 1) / RB;
  const int tile = tiles - 1 - (int)blockIdx.x / nbh;      // causal: the longest rows first
  int b, hk, h;
  split_bh(p, (int)blockIdx.x % nbh, b, hk, h);
  const int row0 = tile * RB, start = uniform(start_of(p, b));
  const int rlast = min(row0 + RB, p.Sq) - 1;
  int kend = uniform(key_limit(p, b));                                 // keys behind it are seen by no row of the block, and not read
  if (p.causal) kend = min(kend, start + rlast + 1);
  const int qrow = row0 + wrow + (lane & 31);
  const bool live = qrow < p.Sq;
  const int qlo = start + row0 + wrow, qhi = qlo + 31, qpos = start + qrow;
  const T* kb = (const T*)p.k + b * p.kb + hk * p.kh;
  const T* vb = (const T*)p.v + b * p.vb + hk * p.vh;
  const T* qp = (const T*)p.q + b * p.qb + h * p.qh + (long long)qrow * p.qs + map * W;
  Frag<T> qf[W / 16];
#pragma unroll
  for (int i = 0; i < W / 16; ++i) qf[i] = frag_global(qp, i, lane, live);
  const float c = positive_scale(p.scale, qf);
  float base = 0.f;
  bool wide = false;
  if (p.bk.n) {
    fill_bias(p, tab, h, tid, 256, false);                             // does not wait for what is hardly ever so
    wide = wide_head(p, h, lane);
    if (wide) {
      fill_bias(p, tab, h, tid, 256, true);
      base = row_base(p, h, qpos, kend);
    }
  }
  f32x16 acc[D / 32];
#pragma unroll
  for (int j = 0; j < D / 32; ++j) acc[j] = zero16();
  float m = -INFINITY, l = 0.f;
  constexpr int ROWS = row_tile<T, D, MAPS>(), NT = sizeof(T) == 2 && D * 2 / MAPS <= 128 ? 1 : ROWS / 32;      // 32-key tiles of one softmax step
  const auto walk = [&](auto wide_rows) __attribute__((always_inline)) {
    Stream<T, D, ROWS> kv(lds);
    if (kend > 0) kv.next(kb, p.ks, vb, p.vs, 0, kend, tid);
    for (int k0 = 0; k0 < kend; k0 += ROWS) {
      kv.arrive();
      if (k0 + ROWS < kend) kv.next(kb, p.ks, vb, p.vs, k0 + ROWS, kend, tid);
#pragma unroll 1
      for (int r0 = 0; r0 < ROWS; r0 += 32 * NT)
        if (k0 + r0 < kend && (!p.causal || k0 + r0 <= qhi))
          tile_step<T, D, ROWS, W, NT, decltype(wide_rows)::value>(p, kv.a(), kv.b(), qf, acc, m, l, c, map, r0, k0 + r0, kend, qpos, qlo, qhi, tab, base,
                                                                   lane);
    }
  };
  if (wide) walk(std::true_type{});        // a loop of its own: the ordinary one pays nothing for it
  else walk(std::false_type{});
  l = column_sum(l);
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int j = 0; j < D / 32; ++j) acc[j] = l == 0.f ? zero16() : acc[j] * inv;      // a row that sees no key: 0 whatever the values hold
  if (p.lse && live && half == 0)
    p.lse[(((size_t)b * p.H + h) * MAPS + map) * p.Sq + qrow] = l > 0.f ? m + __builtin_amdgcn_logf(l) : INFINITY;
  const size_t orow = (((size_t)b * p.Sq + qrow) * p.H + h) * D;
  if constexpr (MAPS == 2) {
    // the second map's rows meet the first's through LDS: [64 rows][D] fp32, one column of 4 floats per lane and register quad
    float* meet = (float*)lds;
    constexpr int MROW = D + 4;
    __syncthreads();
    if (map == 1) {
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d = 32 * j + 8 * g + 4 * half;
          f32x4 v = {acc[j][4 * g], acc[j][4 * g + 1], acc[j][4 * g + 2], acc[j][4 * g + 3]};
          *(f32x4*)(meet + (wrow + (lane & 31)) * MROW + d) = v;
          if (p.out2 && live) store4((T*)p.out2 + orow + d, v[0], v[1], v[2], v[3]);
        }
    }
    __syncthreads();
    if (map == 0 && live) {
      const float lam = ldf(p.lam, h, p.lam_f32);
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d = 32 * j + 8 * g + 4 * half;
          const f32x4 v = *(const f32x4*)(meet + (wrow + (lane & 31)) * MROW + d);
          store4((T*)p.out + orow + d, acc[j][4 * g] - lam * v[0], acc[j][4 * g + 1] - lam * v[1], acc[j][4 * g + 2] - lam * v[2],
                 acc[j][4 * g + 3] - lam * v[3]);
        }
    }
  } else if (live) {
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        store4((T*)p.out + orow + 32 * j + 8 * g + 4 * half, acc[j][4 * g], acc[j][4 * g + 1], acc[j][4 * g + 2], acc[j][4 * g + 3]);
  }
}

// ---- step form ----
// Two maps, bf16: the value products are of A = P_0 - mix P_1 and of P_1, with mix an estimate of lambda l_0 / l_1 (each
// row's own, in the units of its references).  U = sum A v then already is the difference that leaves, its weights rounded once as
// one map's are, and what the rounding of P_1 puts into W = sum P_1 v counts only as far as the estimate is off:
//   sum P_0 v = U + mix W      out = (U + mix W) / l_0 - lambda W / l_1
// (With the maps apart their roundings add up: 4 caches of 8192 .. 32768 keys 2.57e-3 off, now 2.33e-3, which is one map's error
// too; the final rounding alone is 1.66e-3.  80 us either way.)  It begins with a wave's second tile, which has an estimate: on
// a walk of one tile the largest weights, which are 1 and not rounded at all, count for more.  mix is set anew when the references
// move and at tiles 1, 2, 4, 8, ...; a0, a1: the maps' factors then.
template <typename T, int MAPS> constexpr bool mixes() { return MAPS == 2 && sizeof(T) == 2; }
template <int J>
__device__ __forceinline__ void move_mix(f32x16 (&u)[J], f32x16 (&w)[J], float& mix, float a0, float a1, float l0, float l1, float lam) {
  l0 = column_sum(l0);
  l1 = column_sum(l1);
  const float next = l0 > 0.f && l1 > 0.f ? fminf(fmaxf(lam * l0 / l1, -65536.f), 65536.f) : 0.f;       // any finite value is right
  const float k = a0 * mix - a1 * next;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    u[j] = a0 * u[j] + k * w[j];
    w[j] *= a1;
  }
  mix = next;
}
// part (fp32): per (b, key head, row block, split, map): [32 rows][D] unnormalised sums, then per row (maximum, sum)
template <int D, int MAPS> constexpr int part_floats() { return MAPS * 32 * (D + 2); }

// A wave streams its own 32-key tiles (every WAVES-th of the block's chunk) through two private buffers: it waits for its own
// loads only, so no barrier stands between the waves until they meet at the end, and one tile is on its way while one is used.
template <typename T, int D> constexpr int step_waves() { return sizeof(T) * D > 256 ? 2 : 4; }

// runs over all sequences where the registers allow the loop
template <typename T, int D, int MAPS> constexpr bool step_levels() { return !(sizeof(T) == 4 && D == 128 && MAPS == 2); }
// key tiles of a sequence in a step-form call with `level`
__device__ __forceinline__ int step_tiles(const Params& p, int b, int keys) {
  int kend = key_limit(p, b);
  if (p.causal) kend = min(kend, start_of(p, b) + p.Sq);
  return kend > 0 ? (kend + keys - 1) / keys : 0;
}

template <typename T, int D, int MAPS>
__global__ __launch_bounds__((64 * step_waves<T, D>())) void attn_step_kernel(const Params p) {
  using TK = Tile<T, D>;
  constexpr int W = D / MAPS, WAVES = step_waves<T, D>(), T32 = 32 * TK::ROWB;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  char* mine = lds + wave * 4 * T32;                           // two of (K, V)
  constexpr int KEYS = 32 * WAVES, THREADS = 64 * WAVES;
  const bool level = step_levels<T, D, MAPS>() && p.level;
  const int G = p.H / p.Hkv, rows = G * p.Sq, rblocks = (rows + 31) / 32;
  // bias: bucket per distance (one byte) and the key head's columns of the table; two LDS reads per score near the query, the
  // last buckets' values (one pair per query head, so per lane) everywhere else
  unsigned char* ids = (unsigned char*)(lds + WAVES * 4 * T32);
  const int reach = p.bk.reach;
  float* tab = (float*)(ids + (p.bk.n ? ((2 * reach + 1 + 15) & ~15) : 0));
  int* wides = (int*)(tab + p.bk.n * G);                       // [WAVES]: a wave has filled in a wide entry
  int* before = wides + WAVES;
  if (p.bk.n)
    for (int i = tid; i <= 2 * reach; i += THREADS) ids[i] = (unsigned char)bucket_of(p.bk, i - reach);
  // Lengths that differ (level): the key tiles of all sequences and key heads form one line, cut into equal runs, one to a block;
  // a run ends one sequence's part and begins the next where it has to.  Otherwise a block has one split of one row block.
  long long t = 0, t_end = 1;
  if (level) {
    if (wave == 0) {
      int sum = 0;
      for (int b0 = 0; b0 < p.B; b0 += 64) {
        const int b = b0 + lane;
        int n = b < p.B ? step_tiles(p, b, KEYS) : 0, inc = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const int up = __shfl_up(inc, o, 64);
          if (lane >= o) inc += up;
        }
        if (b < p.B) before[b] = sum + inc - n;
        sum += __shfl(inc, 63, 64);
      }
      if (lane == 0) before[p.B] = sum;
    }
    __syncthreads();
    if (blockIdx.x == 0)
      for (int i = tid; i <= p.B; i += THREADS) p.tiles_before[i] = before[i];
    const long long tiles_all = (long long)before[p.B] * p.Hkv;
    const long long runs = min(tiles_all, (long long)gridDim.x);   // no run is empty: every slot that a key head's tiles span is written
    if ((long long)blockIdx.x >= runs) return;
    t = tiles_all * blockIdx.x / runs;
    t_end = tiles_all * (blockIdx.x + 1) / runs;
  }
  for (; t < t_end;) {
  int b, hk, rb = 0, k_lo, k_hi, tiles = 1;
  size_t slot = blockIdx.x;
  if (level) {
    int lo = 0, hi = p.B;                                        // the sequence with before[b] Hkv <= t < before[b + 1] Hkv
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if ((long long)before[mid] * p.Hkv <= t) lo = mid;
      else hi = mid;
    }
    b = __builtin_amdgcn_readfirstlane(lo);
    const int n = __builtin_amdgcn_readfirstlane(before[b + 1] - before[b]), in = (int)(t - (long long)before[b] * p.Hkv);
    hk = __builtin_amdgcn_readfirstlane(in / n);
    const int first = __builtin_amdgcn_readfirstlane(in % n);
    tiles = (int)(t_end - t < n - first ? t_end - t : n - first);
    k_lo = first * KEYS;
    k_hi = (first + tiles) * KEYS;
    slot += b * p.Hkv + hk;
  } else {
    int j = (int)blockIdx.x / p.splits;
    rb = j % rblocks;
    j /= rblocks;
    hk = j % p.Hkv;
    b = j / p.Hkv;
  }
  const int row = rb * 32 + (lane & 31);
  const bool live = row < rows;
  const int g = live ? row / p.Sq : 0, qi = live ? row % p.Sq : 0, h = hk * G + g;
  const int limit = uniform(key_limit(p, b)), start = uniform(start_of(p, b)), qpos = start + qi;
  // positions of the block's first and last query (all of them where its rows reach into a second head)
  const int r_last = min(rows, rb * 32 + 32) - 1;
  const bool one = rb * 32 / p.Sq == r_last / p.Sq;
  const int qlo = start + (one ? rb * 32 % p.Sq : 0), qhi = start + (one ? r_last % p.Sq : p.Sq - 1);
  int kend = limit;
  if (p.causal) kend = max(0, min(kend, qhi + 1));
  if (!level) {      // the splits share the keys that are there, not the cache's length
    const int chunk = ((kend + p.splits - 1) / p.splits + KEYS - 1) / KEYS * KEYS;
    k_lo = (int)blockIdx.x % p.splits * chunk;
    k_hi = k_lo + chunk;
  }
  k_hi = min(kend, k_hi);
  const T* kb = (const T*)p.k + b * p.kb + hk * p.kh;
  const T* vb = (const T*)p.v + b * p.vb + hk * p.vh;
  const T* qp = (const T*)p.q + b * p.qb + h * p.qh + (long long)qi * p.qs;
  int k0 = k_lo + 32 * wave;
  if (k0 < k_hi) {
    TK::dma32(kb, p.ks, k0, k_hi, mine, lane);
    TK::dma32(vb, p.vs, k0, k_hi, mine + T32, lane);
  }
  float far_l = 0.f, far_r = 0.f, base = 0.f;
  if (p.bk.n) {
    bool any = false;
    for (int i = tid; i < p.bk.n * G; i += THREADS) {
      const float v = ldf(p.bias, (size_t)(i / G) * p.H + hk * G + i % G, p.bias_f32);
      any = any || wide_entry(v);
      tab[i] = QUARTER * v;                                        // here always in this unit: a few tiles look entries up
    }
    const bool mine_any = __any(any);
    if (lane == 0) wides[wave] = mine_any;
    __syncthreads();
    any = false;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) any = any || wides[w];
    if (any) {                                                     // only the lanes of the heads that are wide (as wide_head has it)
      bool head = false;
      for (int u = 0; u < p.bk.n; ++u) head = head || wide_entry(ldf(p.bias, (size_t)u * p.H + h, p.bias_f32));
      if (head) base = row_base(p.bk, qpos, min(limit - 1, p.causal ? qpos : 0x7fffffff), [&](int u) { return tab[u * G + g]; });
    }
    far_l = 4.f * (tab[ids[0] * G + g] - base);
    far_r = 4.f * (tab[ids[2 * reach] * G + g] - base);
  }
  Frag<T> qf[D / 16];
#pragma unroll
  for (int i = 0; i < D / 16; ++i) qf[i] = frag_global(qp, i, lane, live);
  f32x16 acc[MAPS][D / 32];
  float m[MAPS], l[MAPS];
#pragma unroll
  for (int a = 0; a < MAPS; ++a) {
    m[a] = -INFINITY;
    l[a] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[a][i] = zero16();
  }
  const float c = positive_scale(p.scale, qf);
  float lam = 0.f, mix = 0.f;
  if constexpr (MAPS == 2) lam = ldf(p.lam, h, p.lam_f32);
  for (int flip = 0; k0 < k_hi; k0 += 32 * WAVES, flip ^= 1) {
    char *wk = mine + flip * 2 * T32, *wv = wk + T32;
    wait_reads();
    if (k0 + 32 * WAVES < k_hi) {
      char* to = mine + (flip ^ 1) * 2 * T32;
      TK::dma32(kb, p.ks, k0 + 32 * WAVES, k_hi, to, lane);
      TK::dma32(vb, p.vs, k0 + 32 * WAVES, k_hi, to + T32, lane);
      wait_dma<2 * TK::PER32>();
    } else {
      wait_dma<0>();
    }
    const bool near = p.bk.n && k0 + 31 - qlo > -reach && k0 - qhi < reach;
    const bool whole = k0 + 31 < k_hi && (!p.causal || k0 + 31 <= qlo);
    const float far = k0 + 31 - qlo <= -reach ? far_l : far_r;
    f32x16 s[MAPS];
    float cc = c, off = far, al[MAPS];
    bool up = false;
#pragma unroll
    for (int a = 0; a < MAPS; ++a) {
      s[a] = zero16();
#pragma unroll
      for (int i = 0; i < W / 16; ++i) s[a] = mma(TK::frag(wk, 0, a * (W / 16) + i, lane), qf[a * (W / 16) + i], s[a]);
    }
    if (near || !whole) {
      const int last = min(k_hi - 1, p.causal ? qpos : 0x7fffffff) - k0 - 4 * half;              // last visible key of this lane's query
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int k = 8 * (r >> 2) + (r & 3);
        float add = far;
        if (near) {
          int rel = k0 + 4 * half + k - qpos;
          rel = rel < -reach ? -reach : (rel > reach ? reach : rel);
          add = 4.f * (tab[ids[rel + reach] * G + g] - base);
        }
#pragma unroll
        for (int a = 0; a < MAPS; ++a) s[a][r] = k > last ? -INFINITY : fmaf(s[a][r], c, add);
      }
      cc = 1.f;
      off = 0.f;
    }
    // as in softmax_tile: the reference follows the maximum in steps of 2^SLACK
#pragma unroll
    for (int a = 0; a < MAPS; ++a) {
      float top = s[a][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = fmaxf(top, s[a][r]);
      al[a] = fmaf(column_max(top), cc, off);
      up = up || al[a] > m[a] + SLACK;
    }
    const bool moved = __any(up);
#pragma unroll
    for (int a = 0; a < MAPS; ++a) {
      const float mn = moved ? fmaxf(m[a], al[a]) : m[a];
      al[a] = 1.f;
      if (moved) {
        al[a] = exp2_(m[a] - (mn == -INFINITY ? 0.f : mn));
        m[a] = mn;
        l[a] *= al[a];
        if constexpr (!mixes<T, MAPS>())
#pragma unroll
          for (int i = 0; i < D / 32; ++i) acc[a][i] *= al[a];
      }
    }
#pragma unroll
    for (int a = 0; a < MAPS; ++a) {
      const float base = off - (m[a] == -INFINITY ? 0.f : m[a]);
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[a][r] = exp2_(fmaf(s[a][r], cc, base));
        sum += s[a][r];
      }
      l[a] += sum;
    }
    if constexpr (mixes<T, MAPS>()) {
      const int n = (k0 - k_lo) / (32 * WAVES);
      if (moved || (n > 0 && (n & (n - 1)) == 0)) move_mix(acc[0], acc[1], mix, al[0], al[1], l[0], l[1], n > 0 ? lam : 0.f);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[0][r] = fmaf(-mix, s[1][r], s[0][r]);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      Frag<T> pf[MAPS];
#pragma unroll
      for (int a = 0; a < MAPS; ++a) to_frag(pf[a], s[a], 8 * u);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const Frag<T> vt = TK::frag_t(wv, 16 * u, 32 * i, lane);
#pragma unroll
        for (int a = 0; a < MAPS; ++a) acc[a][i] = mma(vt, pf[a], acc[a][i]);
      }
    }
  }
  if constexpr (mixes<T, MAPS>())
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[0][i] += mix * acc[1][i];
  // join the waves: [wave][32 rows][D + 4] sums and [wave][32][2] statistics, one map at a time
  constexpr int MROW = D + 4;
  float* meet = (float*)lds;
  float* stat = meet + WAVES * 32 * MROW;
  float* part = p.part + slot * part_floats<D, MAPS>();
  constexpr int ITEMS = 32 * D / 4 / (64 * WAVES);             // 4-column pieces of the [32][D] tile per thread
  f32x4 first[ITEMS];
#pragma unroll
  for (int a = 0; a < MAPS; ++a) {
    __syncthreads();
    const float lt = column_sum(l[a]);
    const int col = lane & 31;
    if (lt == 0.f)                                             // no key of this wave's: 0 whatever the values hold
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[a][i] = zero16();
    if (half == 0) {
      stat[(wave * 32 + col) * 2] = m[a];
      stat[(wave * 32 + col) * 2 + 1] = lt;
    }
    if (live)
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f32x4 v = {acc[a][i][4 * q], acc[a][i][4 * q + 1], acc[a][i][4 * q + 2], acc[a][i][4 * q + 3]};
          *(f32x4*)(meet + (wave * 32 + col) * MROW + 32 * i + 8 * q + 4 * half) = v;
        }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < ITEMS; ++e) {
      const int i = tid + 64 * WAVES * e, r = i / (D / 4), d = 4 * (i % (D / 4)), at = rb * 32 + r;
      if (at >= rows) continue;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) mm = fmaxf(mm, stat[(w * 32 + r) * 2]);
      const float base = mm == -INFINITY ? 0.f : mm;
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
      float ls = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float f = exp2_(stat[(w * 32 + r) * 2] - base);
        ls += f * stat[(w * 32 + r) * 2 + 1];
        sum += f * *(const f32x4*)(meet + (w * 32 + r) * MROW + d);
      }
      if (p.splits > 1) {
        *(f32x4*)(part + (a * 32 + r) * D + d) = sum;
        if (d == 0) {
          part[MAPS * 32 * D + (a * 32 + r) * 2] = mm;
          part[MAPS * 32 * D + (a * 32 + r) * 2 + 1] = ls;
        }
        continue;
      }
      // the whole key axis in this block: the rows leave from here
      const int hr = hk * G + at / p.Sq, qr = at % p.Sq;
      const size_t o_at = (((size_t)b * p.Sq + qr) * p.H + hr) * D + d;
      sum *= ls > 0.f ? 1.f / ls : 0.f;
      if (p.lse && d == 0) p.lse[(((size_t)b * p.H + hr) * MAPS + a) * p.Sq + qr] = ls > 0.f ? mm + __builtin_amdgcn_logf(ls) : INFINITY;
      if (MAPS == 2 && a == 0) {
        first[e] = sum;
        continue;
      }
      if constexpr (MAPS == 2) {
        if (p.out2) store4((T*)p.out2 + o_at, sum[0], sum[1], sum[2], sum[3]);
        const float lam = ldf(p.lam, hr, p.lam_f32);
        sum = first[e] - lam * sum;
      }
      store4((T*)p.out + o_at, sum[0], sum[1], sum[2], sum[3]);
    }
  }
  t += tiles;
  if (t < t_end) __syncthreads();                                  // the next run's tiles come where the sums lie
  }
}

// joins the splits of a row: one block per (b, key head, row); thread = (4 columns, every RUNS-th split), runs joined in order
constexpr int MAX_SPLITS = 1024;
template <typename T, int D, int MAPS> __global__ __launch_bounds__(256) void attn_join_kernel(const Params p) {
  constexpr int LANES = D / 4, RUNS = 256 / LANES, PF = part_floats<D, MAPS>();
  __shared__ float wt[MAX_SPLITS], red[8];
  __shared__ __attribute__((aligned(16))) float sums[RUNS][D];
  const int G = p.H / p.Hkv, rows = G * p.Sq, rblocks = (rows + 31) / 32;
  const int row = (int)blockIdx.x % rows, bk = (int)blockIdx.x / rows, hk = bk % p.Hkv, b = bk / p.Hkv;
  const int tid = threadIdx.x, d = 4 * (tid % LANES), run = tid / LANES, g = row / p.Sq, qi = row % p.Sq, h = hk * G + g;
  size_t first = ((size_t)bk * rblocks + row / 32) * p.splits;
  int splits = p.splits;
  if (p.level) {                 // the runs that touch this key head's tiles: tile x is in run ((x + 1) runs - 1) / tiles
    const long long all = (long long)p.tiles_before[p.B] * p.Hkv, runs = min(all, (long long)p.level), n = p.tiles_before[b + 1] - p.tiles_before[b];
    const long long x = (long long)p.tiles_before[b] * p.Hkv + hk * n;
    const long long i0 = n ? ((x + 1) * runs - 1) / all : 0, i1 = n ? ((x + n) * runs - 1) / all : -1;
    first = (size_t)(i0 + bk);
    splits = (int)(i1 - i0 + 1);
  }
  const float* part = p.part + first * PF;
  f32x4 o[MAPS];
#pragma unroll
  for (int a = 0; a < MAPS; ++a) {
    const float* st = part + MAPS * 32 * D + (a * 32 + row % 32) * 2;
    float ms = -INFINITY;
    for (int s = tid; s < splits; s += 256) ms = fmaxf(ms, st[(size_t)s * PF]);
    ms = wave_max(ms);
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6] = ms;
    __syncthreads();
    const float mm = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), base = mm == -INFINITY ? 0.f : mm;
    float ls = 0.f;
    for (int s = tid; s < splits; s += 256) {
      const float f = exp2_(st[(size_t)s * PF] - base);
      wt[s] = f;
      ls += f * st[(size_t)s * PF + 1];
    }
    ls = wave_sum(ls);
    if ((tid & 63) == 0) red[4 + (tid >> 6)] = ls;
    __syncthreads();
    const float l = (red[4] + red[5]) + (red[6] + red[7]);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int s = run; s < splits; s += RUNS) sum += wt[s] * *(const f32x4*)(part + (size_t)s * PF + (a * 32 + row % 32) * D + d);
    *(f32x4*)(&sums[run][d]) = sum;
    __syncthreads();
    if (run == 0) {
#pragma unroll
      for (int r = 1; r < RUNS; ++r) sum += *(const f32x4*)(&sums[r][d]);
      o[a] = sum * (l > 0.f ? 1.f / l : 0.f);
    }
    if (p.lse && tid == 0) p.lse[(((size_t)b * p.H + h) * MAPS + a) * p.Sq + qi] = l > 0.f ? mm + __builtin_amdgcn_logf(l) : INFINITY;
  }
  if (run) return;
  const size_t at = (((size_t)b * p.Sq + qi) * p.H + h) * D + d;
  if constexpr (MAPS == 2) {
    if (p.out2) store4((T*)p.out2 + at, o[1][0], o[1][1], o[1][2], o[1][3]);
    const float lam = ldf(p.lam, h, p.lam_f32);
    o[0] -= lam * o[1];
  }
  store4((T*)p.out + at, o[0][0], o[0][1], o[0][2], o[0][3]);
}

constexpr int LEVEL_BATCH = 1024;      // sequences whose lengths a block adds up for itself

struct Plan {
  bool step;
  int splits, rblocks, level;            // level: blocks that share the tiles of all sequences, or 0
  size_t lds, part_bytes, before_bytes;
};

template <typename T, int D, int MAPS> Plan plan_of(const Params& p) {
  Plan r{};
  constexpr int WAVES = step_waves<T, D>(), KEYS = 32 * WAVES;
  const long long G = p.H / p.Hkv, rows = G * p.Sq;
  const size_t bias = p.bk.n ? (size_t)((2 * p.bk.reach + 16) & ~15) + 4 * (size_t)p.bk.n * G : 0;
  const size_t meet = (size_t)WAVES * 32 * (D + 4) * 4 + WAVES * 32 * 2 * 4;
  r.lds = WAVES * 4 * 32 * (size_t)Tile<T, D>::ROWB + bias + 4 * WAVES;
  if (r.lds < meet) r.lds = meet;
  // Step form: few rows per key head (then only the key axis can fill the chip), or fewer blocks of the row form than CUs
  r.step = (rows <= 32 || (long long)p.B * p.H * ((p.Sq * (long long)MAPS + 127) / 128) < CUS) && r.lds <= 160 * 1024;
  if (!r.step) return r;
  r.rblocks = (int)((rows + 31) / 32);
  const long long base = (long long)p.B * p.Hkv * r.rblocks, keys = rows <= 32 ? KEYS : SPLIT_KEYS, most = (p.Sk + keys - 1) / keys;
  // one round of blocks: as many as the CUs hold at once (bf16 at 128 columns: one each; 32 ragged caches of 4096 keys 52 us with
  // 256 blocks, 57 with 512, 64 with 1024).  Many rows: joining costs more than a few idle CUs.
  long long each = 160 * 1024 / r.lds, blocks = CUS * (each > 4 ? 4 : each);
  long long want = rows <= 32 ? (blocks + base - 1) / base : CUS / base;
  if (want < 1) want = 1;
  if (want > most) want = most;
  if (want > MAX_SPLITS) want = MAX_SPLITS;
  r.splits = (int)want;
  // Lengths of their own for the sequences: equal runs over all of them (32 caches of 1024 .. 4096 keys: 52 us with two splits
  // each, where the longest cache sets the time; 50 us in runs).
  if (step_levels<T, D, MAPS>() && p.kv_len && rows <= 32 && want > 1 && base * most < (1ll << 30) && p.B <= LEVEL_BATCH && r.lds + 4 * (size_t)(p.B + 1) <= 160 * 1024) {
    r.level = (int)(base * most < blocks ? base * most : blocks);
    r.lds += 4 * (size_t)(p.B + 1);
    r.before_bytes = (4 * (size_t)(p.B + 1) + 15) & ~(size_t)15;
    r.part_bytes = ((size_t)r.level + base) * part_floats<D, MAPS>() * 4 + r.before_bytes;
    return r;
  }
  r.part_bytes = r.splits > 1 ? (size_t)base * r.splits * part_floats<D, MAPS>() * 4 : 0;
  return r;
}

template <typename T, int D, int MAPS> size_t fwd_workspace(const Params& p) { return plan_of<T, D, MAPS>(p).part_bytes; }

template <typename T, int D, int MAPS> int run_fwd(Params& p, void* ws, size_t ws_bytes, hipStream_t st) {
  const char* who = "token_attention_fwd";
  const Plan r = plan_of<T, D, MAPS>(p);
  if (r.step) {
    EOVAE_CHECK_ARG(r.part_bytes == 0 || (ws && ws_bytes >= r.part_bytes), "%s: workspace of %zu bytes, needs %zu", who, ws_bytes, r.part_bytes);
    p.part = (float*)((char*)ws + r.before_bytes);
    p.tiles_before = (int*)ws;
    p.splits = r.splits;
    p.level = r.level;
    const size_t base = (size_t)p.B * p.Hkv;
    const int rc = launch(attn_step_kernel<T, D, MAPS>, r.level ? (size_t)r.level : base * r.rblocks * r.splits, 64 * step_waves<T, D>(), r.lds, p, st, who);
    if (rc || r.splits == 1) return rc;
    return launch(attn_join_kernel<T, D, MAPS>, base * (p.H / p.Hkv) * p.Sq, 256, 0, p, st, who);
  }
  constexpr int RB = 128 / MAPS;
  size_t lds = (size_t)Stream<T, D, row_tile<T, D, MAPS>()>::BYTES + 4 * (size_t)bias_entries(p.bk);
  if (MAPS == 2 && lds < (size_t)64 * (D + 4) * 4) lds = (size_t)64 * (D + 4) * 4;
  return launch(attn_rows_kernel<T, D, MAPS>, (size_t)((p.Sq + RB - 1) / RB) * p.B * p.H, 256, lds, p, st, who);
}

}  // namespace

extern "C" int eovae_token_attention_fwd(const eovae_token_attention* d, void* stream) {
  Params p;
  const int rc = make_params(d, p, "token_attention_fwd", 0);
  if (rc) return rc;
  return TOK_DISPATCH(d, run_fwd, p, d->ws, d->ws_bytes, (hipStream_t)stream);
}

size_t tok_fwd_workspace(const eovae_token_attention* d, const Params& p) { return TOK_DISPATCH(d, fwd_workspace, p); }
