// Shared device code of the token attention kernels (token_attn_fwd.hip, token_attn_bwd.hip).
//
//   S_m = scale * Q_m K_m^T + bias[bucket(key position - query position)][head]      m = 0 (and 1: differential attention)
//   O   = softmax(S_0) V                or        (softmax(S_0) - lambda[head] softmax(S_1)) V
//
// One fragment shape serves every product: v_mfma_f32_32x32x16 on bf16, and for fp32 eight v_mfma_f32_32x32x2 on the SAME
// lane layout (lane l holds row l % 32 and the eight k of its half l / 32; the order of k inside an instruction is free as
// long as both operands agree on it).  The accumulator leaves lane l with column l % 32 and the rows 8 (r / 4) + 4 (l / 32)
// + r % 4, r < 16: eight consecutive registers are a B operand of the next product whose k run {4h..4h+3, 8+4h..8+4h+3}
// (h = l / 32), so probabilities and score gradients go from one product into the next without leaving their lane, as long
// as the A operand is read in that order (frag_t below).
//
// What is rounded to fewer bits than fp32 where the tensors are bf16 (fp32 tensors: nothing).  The matrix instructions that keep up
// take 16-bit operands, so what is formed in between enters the next product as bf16, each value rounded once:
//   unnormalised probabilities, for O (each map's own in the row form; the step form subtracts the maps first);
//   w_0 P_0 + w_1 P_1, subtracted in fp32, for dV;        score gradients, for dQ and dK;
//   O and O_1 as they are stored, for the delta of dQ and the near buckets' bias gradient (of dK too where no row sums are formed).
// Scores, statistics, sums, the difference of two maps and everything the table's far buckets and lambda get stay in fp32.
// Measured against 64 bits (rms, relative; rounding only the result is 1.66e-3): one map's output, dV and dK 2.35e-3, dQ 2.4e-3 (2.7e-3
// on rows of some hundred keys); two maps' output 2.33e-3 in the step form, 2.4e-3 .. 2.55e-3 in the row form.  What exact
// weights would take was measured for two maps: a second product with what the rounding left takes them to 1.9e-3, and 16 x 8 x
// 1024 x 64 from 53 to 69 us; both maps in one wave, subtracted first, to 2.34e-3, and 16 x 1000 x 8 x 128 from 108 to 133.
#pragma once
#include <math.h>
#include "eovae_common.h"
#include "../../include/eovae_hip.h"

namespace tok {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int MAX_BUCKETS = 128;       // per side: at most 64 borders behind the exact half
constexpr int MAX_REACH = 1024;
constexpr int TILE = 64;               // rows of a staged tile (Tile::ROWS), at most
constexpr int PAD = 32 + TILE;         // a 32 x TILE tile that touches |rel| < reach stays inside [-reach - PAD, reach + PAD]

// Buckets of one side: n < exact -> n, else exact + #{borders <= n}.  reach: first distance of the last bucket (everything
// at and behind it shares one value).  two_sided: positive distances use the second half of the table.
struct Buckets {
  int n, side, exact, nborders, reach, two_sided;
  int border[MAX_BUCKETS / 2];
};

__device__ __forceinline__ int bucket_of(const Buckets& t, int rel) {
  int n = t.two_sided ? (rel < 0 ? -rel : rel) : (rel < 0 ? -rel : 0);
  int b = n;
  if (n >= t.exact) {
    b = t.exact;
    for (int i = 0; i < t.nborders; i += 8)       // border[] is padded with the largest int: eight at a time, one scalar load
#pragma unroll
      for (int j = 0; j < 8; ++j) b += n >= t.border[i + j] ? 1 : 0;
  }
  return b + (t.two_sided && rel > 0 ? t.side : 0);
}

struct Params {
  const void *q, *k, *v, *o2, *d_o, *o;
  void *out, *out2;
  void *dq, *dk, *dv;
  const void *bias, *lam;
  const int *kv_len, *q_start;
  float *dk_part, *dv_part;                   // [parts] of dk and dv in fp32, where a block walks only a part of the queries
  float *lse, *delta, *part, *lam_part;      // lse: [B][H][maps][Sq], log2 domain, relative to the row's base (+inf: nothing visible); delta likewise
  float* base;                                // backward, from dQ to dK/dV: [B][H][Sq], rows of wide heads
  int* wide;                                  // [H]
  long long qb, qs, qh, kb, ks, kh, vb, vs, vh;   // element strides: batch, token, head
  int B, Sq, Sk, H, Hkv, start, causal, bias_f32, lam_f32, splits, parts, level;
  int* tiles_before;                          // [B + 1], step form with `level`: key tiles of the sequences before each
  float scale;
  Buckets bk;
};

template <typename T> struct Frag;
template <> struct Frag<__bf16> { bf16x8 x; };
template <> struct Frag<float> { f32x8 x; };

__device__ __forceinline__ f32x16 mma(const Frag<__bf16>& a, const Frag<__bf16>& b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.x, b.x, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(const Frag<float>& a, const Frag<float>& b, f32x16 c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x[i], b.x[i], c, 0, 0, 0);
  return c;
}

__device__ __forceinline__ float ldf(const void* p, size_t i, int is_f32) {
  return is_f32 ? ((const float*)p)[i] : (float)((const __bf16*)p)[i];
}
// A finite bias beyond WIDE (the type's lowest value as a mask, say) would swallow the scores that it is added to, and the logarithm
// of a row's sum beside it; yet a query that sees nothing else still has a softmax.  A head with such an entry is `wide`: its
// rows are worked on relative to their `base`, the largest bias among the keys that the row sees (row_base; a softmax does not
// see a constant), and its table is held in QUARTER units of log 2, so that no entry and no difference of two leaves fp32.
// Other heads have base 0; they are walked by loops of their own and pay nothing per score.
constexpr float WIDE = 88.f, QUARTER = 0.25f * LOG2E;        // 88: about 2^7 in units of log 2, where lse still resolves 2^-16
__device__ __forceinline__ bool wide_entry(float v) { return fabsf(v) > WIDE && fabsf(v) < INFINITY; }

// 16 bytes per lane from `src` to LDS at `to` + 16 * lane.  The compiler does not count it: wait_dma() does.
__device__ __forceinline__ void load_lds16(const void* src, unsigned to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(src) : "memory", "m0");
}
// a pointer that is the same in every lane, in scalar registers
__device__ __forceinline__ const char* scalar(const void* p) {
  const unsigned long long v = (unsigned long long)p;
  return (const char*)(((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
                       (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)v));
}
// the same from a wave-uniform address and 32 bits of the lane's own: no vector instruction per load
__device__ __forceinline__ void load_lds16(const void* base, unsigned off, unsigned to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory", "m0");
}
// until at most N of the wave's newest loads are still on their way
template <int N> __device__ __forceinline__ void wait_dma() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// the wave's LDS reads are done: what they read may be overwritten
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// ---- staged tiles: ROWS rows of D elements, 16-byte chunks, chunk index XORed with swz(row) ----
// Eight consecutive rows at one chunk index (a fragment read: lanes = rows) fall into eight different 16-byte bank groups,
// and four consecutive rows times two consecutive chunks (a transposed 16-bit read) cover all 128 bytes once.
// default rows; fp32 rows of 128: half, so that two pairs of tiles and the sums fit in LDS
template <typename T, int D> constexpr int tile_rows() { return sizeof(T) * D > 256 ? 32 : TILE; }
template <typename T, int D, int R = tile_rows<T, D>()> struct Tile {
  static constexpr int ROWS = R;
  static constexpr int ROWB = D * (int)sizeof(T);
  static constexpr int CH = ROWB / 16;                       // chunks per row: 4 .. 32
  static constexpr int BYTES = ROWS * ROWB;
  static constexpr int PER = ROWS * CH / 256;                // chunks per thread of a 256-thread block (1 .. 4)
  static __device__ __forceinline__ int swz(int row) {
    return CH >= 8 ? (((row & 3) << 1) | ((row >> 2) & 1)) : ((row & 2) | ((row >> 2) & 1));
  }
  static __device__ __forceinline__ int at(int row, int chunk) { return row * ROWB + ((chunk ^ swz(row)) << 4); }

  // Rows row0 .. row0 + ROWS - 1 of a strided matrix straight into LDS (global_load_lds: a wave's 64 chunks of 16 bytes land one
  // behind the other from the address in M0, so the swizzle is in what a lane ASKS for; 256 / CH rows further down it is the
  // same).  Rows at and behind `limit` (>= 1) become copies of row limit - 1: finite wherever the caller's data is, and never
  // visible.  A block of 256 threads calls; wait_dma<0>() before the barrier that publishes it.
  static __device__ __forceinline__ void dma(const T* base, long long stride, int row0, int limit, const char* lds, int tid) {
    int t = tid;
    asm volatile("" : "+v"(t));                 // what follows is cheaper than the registers that would keep it from tile to tile
    const int row = t / CH, col = ((t % CH) ^ swz(row)) << 4;
    const unsigned to = (unsigned)__builtin_amdgcn_readfirstlane((int)((unsigned)(size_t)(__attribute__((address_space(3))) const char*)lds +
                                                                       (unsigned)(tid & ~63) * 16u));
    if (row0 + ROWS <= limit && stride < (1ll << 31) / (long long)(sizeof(T) * ROWS)) {
      const char* src = scalar(base + (long long)row0 * stride);
      const unsigned off = (unsigned)row * (unsigned)(stride * (long long)sizeof(T)) + (unsigned)col;
#pragma unroll
      for (int i = 0; i < PER; ++i) load_lds16(src + (long long)i * (256 / CH) * stride * (long long)sizeof(T), off, to + 4096u * i);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int r = row0 + row + i * (256 / CH);
        load_lds16((const char*)(base + (long long)(r < limit ? r : limit - 1) * stride) + col, to + 4096u * i);
      }
    }
  }
  // 32 rows by one wave for itself alone (32 CH / 64 loads): no barrier, only wait_dma
  static constexpr int PER32 = 32 * CH / 64;
  static __device__ __forceinline__ void dma32(const T* base, long long stride, int row0, int limit, const char* lds, int lane) {
    const unsigned to = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(size_t)(__attribute__((address_space(3))) const char*)lds);
    int l = lane;
    asm volatile("" : "+v"(l));
    if (row0 + 32 <= limit && stride < (1ll << 31) / (long long)(sizeof(T) * 32)) {
      // 64 / CH rows a load; the swizzle repeats after eight rows, so after PHASES loads
      constexpr int STEP = 64 / CH, PHASES = STEP >= 8 ? 1 : 8 / STEP;
      const unsigned line = (unsigned)(stride * (long long)sizeof(T));
      const char* src = scalar(base + (long long)row0 * stride);
#pragma unroll
      for (int f = 0; f < PHASES; ++f) {
        const unsigned off = (unsigned)(l / CH) * line + (unsigned)(((l % CH) ^ swz(l / CH + f * STEP)) << 4);
#pragma unroll
        for (int i = f; i < PER32; i += PHASES) load_lds16(src + (long long)i * STEP * line, off, to + 1024u * i);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < PER32; ++i) {
      const int c = l + 64 * i, row = c / CH, r = row0 + row;
      load_lds16((const char*)(base + (long long)(r < limit ? r : limit - 1) * stride) + (((c % CH) ^ swz(row)) << 4), to + 1024u * i);
    }
  }
  // operand fragment: lane holds row (row0 + l % 32), columns 16 s + 8 (l / 32) .. + 7
  static __device__ __forceinline__ Frag<T> frag(const char* lds, int row0, int s, int lane) {
    const int row = row0 + (lane & 31), half = lane >> 5;
    Frag<T> f;
    if constexpr (sizeof(T) == 2) {
      f.x = *(const bf16x8*)(lds + at(row, 2 * s + half));
    } else {
      const f32x4 a = *(const f32x4*)(lds + at(row, 4 * s + 2 * half)), b = *(const f32x4*)(lds + at(row, 4 * s + 2 * half + 1));
      f.x = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return f;
  }
  // transposed operand: lane holds COLUMN col0 + l % 32 and the rows row0 + {4h .. 4h + 3, 8 + 4h .. 8 + 4h + 3}
  static __device__ __forceinline__ Frag<T> frag_t(char* lds, int row0, int col0, int lane) {
    Frag<T> f;
    const int half = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      // ds_read_b64_tr_b16: each 16-lane group hands in four rows of 16 columns (lane: row l / 4, columns 4 (l % 4)) and
      // gets back, per lane, its column's four rows
      const int g = (lane >> 4) & 1, row = row0 + 4 * half + ((lane & 15) >> 2), col = col0 + 16 * g + 4 * (lane & 3);
      typedef __attribute__((address_space(3))) s16x4 lds4;
      const int off = (col & 7) * 2;
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(lds + at(row, col >> 3) + off));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(lds + at(row + 8, col >> 3) + off));
      f.x = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const int col = col0 + (lane & 31);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = row0 + 4 * half + (i & 3) + 8 * (i >> 2);
        f.x[i] = *(const float*)(lds + at(row, col >> 2) + (col & 3) * 4);
      }
    }
    return f;
  }
};

// Two row streams (keys and values, or queries and upstream gradients) through LDS, one tile of each at a time: two buffers,
// the next pair arrives by DMA while this one is used, one barrier per tile.
//   next(...)      request a pair of tiles
//   arrive()       they are in LDS for every wave: a(), b() until the next arrive; the pair before is free
template <typename T, int D, int R = tile_rows<T, D>()> struct Stream {
  using TK = Tile<T, D, R>;
  static constexpr int BYTES = 4 * TK::BYTES;
  char* lds;
  int flip;
  __device__ __forceinline__ explicit Stream(char* l) : lds(l), flip(0) {}
  __device__ __forceinline__ char* a() const { return lds + flip * 2 * TK::BYTES; }
  __device__ __forceinline__ char* b() const { return a() + TK::BYTES; }
  __device__ __forceinline__ void next(const T* pa, long long sa, const T* pb, long long sb, int row0, int limit, int tid) {
    char* to = lds + (flip ^ 1) * 2 * TK::BYTES;
    TK::dma(pa, sa, row0, limit, to, tid);
    TK::dma(pb, sb, row0, limit, to + TK::BYTES, tid);
  }
  __device__ __forceinline__ void arrive() {
    wait_dma<0>();
    __syncthreads();
    flip ^= 1;
  }
};

// Where a 32-row tile's fragments come from: a staged tile, or (fp32) memory itself, rows at and behind `limit` as row limit - 1
template <typename T, int D, int R = tile_rows<T, D>()> struct Staged {
  char* lds;
  int row, lane;
  __device__ __forceinline__ Frag<T> frag(int r, int s) const { return Tile<T, D, R>::frag(lds, row + r, s, lane); }
  __device__ __forceinline__ Frag<T> frag_t(int r, int col) const { return Tile<T, D, R>::frag_t(lds, row + r, col, lane); }
};
struct InMemory {
  const float* base;
  long long stride;
  int row, limit, lane;
  __device__ __forceinline__ const float* at(int r) const { return base + (long long)(row + r < limit ? row + r : limit - 1) * stride; }
  __device__ __forceinline__ Frag<float> frag(int r, int s) const {
    const float* p = at(r + (lane & 31)) + 16 * s + 8 * (lane >> 5);
    const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
    Frag<float> f;
    f.x = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return f;
  }
  __device__ __forceinline__ Frag<float> frag_t(int r, int col) const {
    Frag<float> f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f.x[i] = at(r + 4 * (lane >> 5) + (i & 3) + 8 * (i >> 2))[col + (lane & 31)];
    return f;
  }
};

// fragment of a row straight from global memory (row < limit, else zero)
template <typename T> __device__ __forceinline__ Frag<T> frag_global(const T* row, int s, int lane, bool ok) {
  Frag<T> f;
  const int c = 16 * s + 8 * (lane >> 5);
#pragma unroll
  for (int i = 0; i < 8; ++i) f.x[i] = (T)0.f;
  if (ok) {
    if constexpr (sizeof(T) == 2) {
      f.x = *(const bf16x8*)(row + c);
    } else {
      const f32x4 a = *(const f32x4*)(row + c), b = *(const f32x4*)(row + c + 4);
      f.x = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  return f;
}

// A negative scale is carried by one operand, and a scale of 0 becomes the smallest number: the largest product is the largest
// score, and a masked -infinity stays one.  (In units of log 2.)
template <typename T, int N> __device__ __forceinline__ float positive_scale(float scale, Frag<T> (&qf)[N]) {
  if (scale < 0.f)
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) qf[i].x[e] = -qf[i].x[e];
  return fmaxf(fabsf(scale) * LOG2E, 1.2e-38f);
}

// eight consecutive accumulator registers as the B operand of the next product
__device__ __forceinline__ void to_frag(Frag<__bf16>& f, const f32x16& a, int r0) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f.x[i] = (__bf16)a[r0 + i];
}
__device__ __forceinline__ void to_frag(Frag<float>& f, const f32x16& a, int r0) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f.x[i] = a[r0 + i];
}

template <typename T> __device__ __forceinline__ void store4(T* p, float a, float b, float c, float d);
template <> __device__ __forceinline__ void store4<__bf16>(__bf16* p, float a, float b, float c, float d) {
  bf16x4 v = {(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)d};
  *(bf16x4*)p = v;
}
template <> __device__ __forceinline__ void store4<float>(float* p, float a, float b, float c, float d) {
  f32x4 v = {a, b, c, d};
  *(f32x4*)p = v;
}

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}
__device__ __forceinline__ int acc_row(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }
// a column's two halves (lanes l and l + 32) together: v_permlane32_swap hands every lane both values
struct Halves { float lo, hi; };
__device__ __forceinline__ Halves halves(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned a = r[0], b = r[1];
  return {__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
__device__ __forceinline__ float column_sum(float x) { const Halves h = halves(x); return h.lo + h.hi; }
__device__ __forceinline__ float column_max(float x) { const Halves h = halves(x); return fmaxf(h.lo, h.hi); }
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ int key_limit(const Params& p, int b) {
  if (!p.kv_len) return p.Sk;
  const int n = p.kv_len[b];
  return n < 0 ? 0 : (n > p.Sk ? p.Sk : n);
}
// position of query row 0 among the keys; clamped so that differences of positions stay inside 32 bits
__device__ __forceinline__ int start_of(const Params& p, int b) {
  const int s = p.q_start ? p.q_start[b] : p.start;
  return s < -(1 << 30) ? -(1 << 30) : (s > (1 << 30) ? (1 << 30) : s);
}

// a value that is the same in every lane, in a scalar register
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// head's bias by distance, log2 domain (wide: QUARTER units): tab[rel + reach + PAD], rel in [-reach - PAD, reach + PAD]
__device__ __forceinline__ void fill_bias(const Params& p, float* tab, int head, int tid, int nthreads, bool wide) {
  const int span = p.bk.reach + PAD;
  const float unit = wide ? QUARTER : LOG2E;
  for (int i = tid; i <= 2 * span; i += nthreads)
    tab[i] = unit * ldf(p.bias, (size_t)bucket_of(p.bk, i - span) * p.H + head, p.bias_f32);
}
// one head's column of the table has a wide entry; the same in every lane of a wave
__device__ __forceinline__ bool wide_head(const Params& p, int head, int lane) {
  bool any = false;
  for (int u = lane; u < p.bk.n; u += 64) any = any || wide_entry(ldf(p.bias, (size_t)u * p.H + head, p.bias_f32));
  return __any(any);
}
// wide heads are rare: few LDS reads in flight, so that their path costs the ordinary one no registers
__device__ __forceinline__ void few_at_a_time() { asm volatile("" ::: "memory"); }
// the first distance of a side's bucket i
__device__ __forceinline__ int first_distance(const Buckets& t, int i) { return i <= t.exact ? i : t.border[i - t.exact - 1]; }
// largest of value(bucket) over the keys 0 .. last that a query at position qpos sees; 0 where there is none, or it is not finite
template <typename V> __device__ __forceinline__ float row_base(const Buckets& t, int qpos, int last, V value) {
  const int r0 = -qpos, r1 = last - qpos;                          // their distances key - query
  float top = -INFINITY;
#pragma unroll 1
  for (int u = 0; u < t.n && last >= 0; ++u) {
    const bool right = t.two_sided && u >= t.side;
    const int i = right ? u - t.side : u, a = right && i == 0 ? 1 : first_distance(t, i);
    const bool open = i == t.side - 1;                             // the last bucket has no end
    const int z = open ? 0 : first_distance(t, i + 1) - 1;         // distances a .. z
    if (!open && z < a) continue;
    const bool ahead = !t.two_sided && i == 0 && r1 >= 0;          // one-sided: keys ahead count as distance 0
    const bool seen = right ? r1 >= a && (open || r0 <= z) : (r0 <= -a && (r1 >= -a || open || r1 >= -z)) || ahead;
    if (seen) top = fmaxf(top, value(u));
  }
  return fabsf(top) < INFINITY ? top : 0.f;
}
// the same from the table in memory, for a query of a wide head that sees keys below `kend`
__device__ __forceinline__ float row_base(const Params& p, int head, int qpos, int kend) {
  return row_base(p.bk, qpos, min(kend - 1, p.causal ? qpos : 0x7fffffff), [&](int u) { return QUARTER * ldf(p.bias, (size_t)u * p.H + head, p.bias_f32); });
}
static inline int bias_entries(const Buckets& b) { return b.n ? 2 * (b.reach + PAD) + 1 : 0; }

// heads that share key heads sit next to each other in launch order with stride B * Hkv: with B * Hkv a multiple of 8 the
// blocks that read one key head land on one XCD and its L2 (workgroups go round the XCDs in launch order)
__device__ __forceinline__ void split_bh(const Params& p, int j, int& b, int& hk, int& h) {
  const int n = p.B * p.Hkv, g = j / n, r = j % n;
  b = r / p.Hkv;
  hk = r % p.Hkv;
  h = hk * (p.H / p.Hkv) + g;
}

// ---- host side ----
// checks a descriptor and turns it into kernel parameters; null pointers are allowed only where the header says so
static inline int make_params(const eovae_token_attention* d, Params& p, const char* who, int backward) {
  EOVAE_CHECK_ARG(d != nullptr, "%s: null descriptor", who);
  EOVAE_CHECK_ARG(d->dtype == EOVAE_F32 || d->dtype == EOVAE_BF16, "%s: dtype %d (0 fp32, 1 bf16)", who, d->dtype);
  EOVAE_CHECK_ARG(d->maps == 1 || d->maps == 2, "%s: %d softmax maps (1 or 2)", who, d->maps);
  EOVAE_CHECK_ARG(d->dim == 64 || d->dim == 128 || (d->dim == 32 && d->maps == 1), "%s: head width %d with %d map(s) (32, 64 or 128; two maps: 64 or 128)",
                  who, d->dim, d->maps);
  EOVAE_CHECK_ARG(d->batch >= 1 && d->sq >= 1 && d->sk >= 1 && d->heads >= 1 && d->kv_heads >= 1 && d->sq <= (1 << 28) && d->sk <= (1 << 28) &&
                      d->batch <= (1 << 20) && d->heads <= (1 << 16),
                  "%s: batch %d, queries %d, keys %d, heads %d / %d out of range", who, d->batch, d->sq, d->sk, d->heads, d->kv_heads);
  EOVAE_CHECK_ARG(d->heads % d->kv_heads == 0, "%s: %d heads over %d key heads", who, d->heads, d->kv_heads);
  const long long es = d->dtype == EOVAE_F32 ? 4 : 2;
  const long long* st[3] = {d->q_strides, d->k_strides, d->v_strides};
  for (int i = 0; i < 3; ++i)
    for (int j = 0; j < 3; ++j)
      EOVAE_CHECK_ARG(st[i][j] >= 0 && st[i][j] * es % 16 == 0, "%s: stride %lld is negative or no multiple of 16 bytes", who, st[i][j]);
  const void* ptrs[] = {d->q, d->k, d->v, d->out, d->out2, d->d_out, d->dq, d->dk, d->dv, d->ws};
  for (const void* x : ptrs) EOVAE_CHECK_ARG((size_t)x % 16 == 0, "%s: a tensor is not 16-byte aligned", who);
  EOVAE_CHECK_ARG(d->q && d->k && d->v && d->out, "%s: null q, k, v or out", who);
  EOVAE_CHECK_ARG(d->maps == 1 || d->lam, "%s: two maps need lambda", who);
  EOVAE_CHECK_ARG(!d->bias || d->bias_dtype == EOVAE_F32 || d->bias_dtype == EOVAE_BF16, "%s: bias dtype %d (0 fp32, 1 bf16)", who, d->bias_dtype);
  EOVAE_CHECK_ARG(!d->lam || d->lam_dtype == EOVAE_F32 || d->lam_dtype == EOVAE_BF16, "%s: lambda dtype %d (0 fp32, 1 bf16)", who, d->lam_dtype);
  EOVAE_CHECK_ARG(isfinite(d->scale), "%s: scale is not finite", who);
  if (backward) {
    EOVAE_CHECK_ARG(d->lse && d->d_out && d->dq && d->dk && d->dv, "%s: null lse, d_out, dq, dk or dv", who);
    EOVAE_CHECK_ARG(d->maps == 1 || d->out2, "%s: two maps need out2 of the forward", who);
    EOVAE_CHECK_ARG(!d->dbias || d->bias, "%s: dbias without a bias table", who);
    EOVAE_CHECK_ARG(!d->dlam || d->maps == 2, "%s: dlam with one map", who);
  }
  p.q = d->q; p.k = d->k; p.v = d->v; p.o2 = d->out2; p.o = d->out; p.d_o = d->d_out;
  p.out = d->out; p.out2 = d->out2;
  p.dq = d->dq; p.dk = d->dk; p.dv = d->dv;
  p.bias = d->bias; p.lam = d->lam;
  p.kv_len = d->kv_len; p.q_start = d->query_start;
  p.lse = d->lse; p.delta = nullptr; p.base = nullptr; p.wide = nullptr; p.part = nullptr; p.lam_part = nullptr;
  p.qb = d->q_strides[0]; p.qs = d->q_strides[1]; p.qh = d->q_strides[2];
  p.kb = d->k_strides[0]; p.ks = d->k_strides[1]; p.kh = d->k_strides[2];
  p.vb = d->v_strides[0]; p.vs = d->v_strides[1]; p.vh = d->v_strides[2];
  p.B = d->batch; p.Sq = d->sq; p.Sk = d->sk; p.H = d->heads; p.Hkv = d->kv_heads; p.start = d->start; p.causal = d->causal ? 1 : 0;
  p.bias_f32 = d->bias_dtype == EOVAE_F32; p.lam_f32 = d->lam_dtype == EOVAE_F32;
  p.splits = 1; p.level = 0; p.tiles_before = nullptr; p.parts = 1; p.dk_part = p.dv_part = nullptr;
  p.scale = d->scale;
  Buckets& t = p.bk;
  t.n = t.side = t.exact = t.nborders = t.reach = t.two_sided = 0;
  for (int& e : t.border) e = 0x7fffffff;
  if (d->bias) {
    EOVAE_CHECK_ARG(d->buckets >= 2 && d->buckets <= MAX_BUCKETS, "%s: %d buckets (2 .. %d)", who, d->buckets, MAX_BUCKETS);
    t.n = d->buckets;
    t.two_sided = d->two_sided ? 1 : 0;
    t.side = t.two_sided ? t.n / 2 : t.n;
    EOVAE_CHECK_ARG(t.side >= 2 && (!t.two_sided || t.n % 2 == 0), "%s: %d buckets over %d side(s)", who, t.n, t.two_sided + 1);
    t.exact = t.side / 2;
    t.nborders = t.side - t.exact - 1;
    EOVAE_CHECK_ARG(t.nborders == 0 || d->borders, "%s: null borders", who);
    t.reach = t.exact;
    for (int i = 0; i < t.nborders; ++i) {
      EOVAE_CHECK_ARG(d->borders[i] >= t.reach && d->borders[i] <= MAX_REACH, "%s: border %d of %d falls, or lies beyond %d", who, i, t.nborders, MAX_REACH);
      t.border[i] = t.reach = d->borders[i];
    }
  }
  return EOVAE_OK;
}

// more than 64 KiB of LDS per block has to be asked for
template <typename K> static inline int launch(K kernel, size_t blocks, int threads, size_t lds, const Params& p, hipStream_t st, const char* who) {
  EOVAE_CHECK_ARG(blocks <= 0x7fffffff, "%s: %zu blocks", who, blocks);
  EOVAE_CHECK_ARG(lds <= 160 * 1024, "%s: %zu bytes of LDS", who, lds);
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) {
      eovae_set_error("%s: %zu bytes of LDS refused: %s", who, lds, hipGetErrorString(e));
      return EOVAE_ERR_LAUNCH;
    }
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), lds, st, p);
  EOVAE_CHECK_LAUNCH(who);
  return EOVAE_OK;
}

}  // namespace tok

// calls F<T, D, MAPS>(args...) for the descriptor's type, width and maps (make_params has checked the combination)
#define TOK_DISPATCH(d, F, ...)                                                                                          \
  ((d)->dtype == EOVAE_F32                                                                                              \
       ? ((d)->maps == 2 ? ((d)->dim == 64 ? F<float, 64, 2>(__VA_ARGS__) : F<float, 128, 2>(__VA_ARGS__))               \
                         : ((d)->dim == 32 ? F<float, 32, 1>(__VA_ARGS__)                                                \
                                           : (d)->dim == 64 ? F<float, 64, 1>(__VA_ARGS__) : F<float, 128, 1>(__VA_ARGS__))) \
       : ((d)->maps == 2 ? ((d)->dim == 64 ? F<__bf16, 64, 2>(__VA_ARGS__) : F<__bf16, 128, 2>(__VA_ARGS__))             \
                         : ((d)->dim == 32 ? F<__bf16, 32, 1>(__VA_ARGS__)                                               \
                                           : (d)->dim == 64 ? F<__bf16, 64, 1>(__VA_ARGS__) : F<__bf16, 128, 1>(__VA_ARGS__))))
