// Cross attention of queries to encoder states of another length, bf16 / fp16, fp32 accumulation, any head dimension that 8 divides up to
// 128, grouped heads (G = Hq / Hk query heads share a key head), a length per sample and a mask:
//     o_r = sum_j p_rj v_j,  p_rj = exp(s_rj - lse_r),  s_rj = scale q_r . k_j,  over the keys j < length[b] that are not blocked
//     dv_j = sum_r p_rj do_r,  ds_rj = p_rj (do_r . v_j - do_r . o_r),  dq_r = scale sum_j ds_rj k_j,  dk_j = scale sum_r ds_rj q_r
// A row without an open key gives zeros and passes no gradient.
//
// Rows: the G query heads of a key head are packed as rows r = query * G + head, so a single token of a grouped model fills a tile with the
// heads that read the same keys.  All products run on v_mfma_f32_32x32x16: score tiles are computed TRANSPOSED (keys x rows), so a lane owns
// one row - the softmax statistics are lane-local plus one exchange with the other half wave - and the tile is, register for register, the B
// operand of the product that follows when that product's contraction runs in the order in which a lane holds its keys (4 h + 0..3,
// 8 + 4 h + 0..3 of every 16).  The A operand in that order is the transpose of a row-major LDS tile: ds_read_b64_tr_b16 reads it, so K, V, Q
// and dO are each staged once, row-major, for both uses.  LDS tiles are padded (Tile).
#include <cmath>
#include <type_traits>

#include "combo_common.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Type;
template <> struct Type<__bf16> {
  typedef bf16x8 x8;
  typedef bf16x4 x4;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Type<_Float16> {
  typedef f16x8 x8;
  typedef f16x4 x4;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

constexpr float kInf = __builtin_huge_valf();

struct Args {
  const char *q, *k, *v;
  long long qb, qn, qh, kb, kn, kh, vb, vn, vh;  // strides in elements
  const int* lens;
  const unsigned* bits;
  long long mb, mh, mn;  // strides of the packed mask in words
  int B, Lq, Lk, Hq, Hk, G, D, rows;
  float scale, c;        // c = scale * log2(e)
  int tiles, splits;
  void* out;             // forward: o; backward: dq (dk, dv below)
  float* lse;            // [B][Hk][rows], base 2; +inf: no open key
  float *part, *part_lse;
  const void *o, *dout;
  float* delta;
  void *dk, *dv;
};

__device__ __forceinline__ int length_of(const Args& A, int b) {
  return A.lens ? min(max(A.lens[b], 0), A.Lk) : A.Lk;
}

// row-major LDS tile of 16-bit values.  The pitch is an odd number p of 16-byte chunks with p = 3, 7 or 9 (mod 16): 16 rows at the same chunk (a
// b128 operand read) start in 16 different chunks of the 64 banks, and 4 rows x 2 neighbouring chunks (16 lanes of a transposed read) in 8, and
// every address is one lane register plus an immediate.  Conflicts are left in a quarter of the LDS cycles (SQ_LDS_BANK_CONFLICT over
// SQ_LDS_IDX_ACTIVE at 64 x 4096 x 4096 x 128: 0.25 forward and dk / dv, 0.20 dq); a swizzle by exclusive-or has none, but costs a register or an
// instruction per operand, of which the kernels are short: forward at that size 1272 us with the swizzle, 997 with the pitch.
template <int DP>
struct Tile {
  static constexpr int PITCH = DP == 32 ? 56 : (DP == 64 ? 72 : 152);
  static __device__ __forceinline__ int at(int r, int c) { return r * PITCH + c * 8; }
};

// A (or B) operand of a product over the row's own dimension: row r0 + (lane & 31), values 16 step + 8 half .. + 7
template <typename T, int DP>
__device__ __forceinline__ typename Type<T>::x8 operand(const T* tile, int r0, int step) {
  const int lane = threadIdx.x & 63;
  return *reinterpret_cast<const typename Type<T>::x8*>(tile + Tile<DP>::at(r0 + (lane & 31), 2 * step + (lane >> 5)));
}

// A operand of a product over the tile's ROWS: value d0 + (lane & 31) of rows r0 + 4 h + 0..3 and r0 + 8 + 4 h + 0..3
template <typename T, int DP>
__device__ __forceinline__ typename Type<T>::x8 operand_t(const T* tile, int r0, int d0) {
  const int lane = threadIdx.x & 63, row = r0 + 4 * (lane >> 5) + ((lane & 15) >> 2);
  const int col = d0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  typedef __attribute__((address_space(3))) s16x4 lds4;
  const T* a = tile + row * Tile<DP>::PITCH + col;
  const T* b = a + 8 * Tile<DP>::PITCH;
  const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)a), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)b);
  return __builtin_bit_cast(typename Type<T>::x8, (s16x8)__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
}

// 8 of a tile's 16 registers as the B operand of the product that follows (values 16 s .. 16 s + 15 of the contraction)
template <typename T>
__device__ __forceinline__ typename Type<T>::x8 pack(const f32x16& p, int s) {
  f32x8 x;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = p[8 * s + i];
  return __builtin_convertvector(x, typename Type<T>::x8);
}

// what pack left off, itself rounded
template <typename T>
__device__ __forceinline__ typename Type<T>::x8 left_off(const f32x16& p, int s, const typename Type<T>::x8& packed) {
  f32x8 x;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = p[8 * s + i] - (float)packed[i];
  return __builtin_convertvector(x, typename Type<T>::x8);
}

__device__ __forceinline__ float other_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// fp16 holds 30 binades, and a score gradient ds = p (dp - delta) carries the size of a probability (1 / keys) times that of the upstream gradient:
// rounded as it is, ds of 16384 keys under upstream gradients of 2^-10 lay below 2^-24, and dq was off by 16 times its own rounding.  So a lane holds
// its row (dq) or key (dk) of ds, and its accumulators, at 2^up and takes that out again at the end.  `up` starts high and only falls: where a value of
// a tile reaches 2, the lane's largest is brought into [2^-7, 2^-6) and the accumulators follow, at the first tile and a few times at most behind it.
// What then lies under 2^-14 is rounded by at most 2^-25, 1/64 of the largest's own rounding, and ds past 65504 stay in range.  bf16 has fp32's
// exponents and holds ds as it is.  Cost in fp16: 4 x 16 x 4096 x 4096 x 128, training, 3035 -> 3254 us; 4 x 10 x 4096 rows against 77 keys 85 -> 87.
struct Held {
  float up = 60.f;
  static __device__ __forceinline__ float power(float e) { return __builtin_amdgcn_ldexpf(1.f, (int)e); }
  // top: this lane's largest |x| -> the factor that x and the accumulators of its row or key, which two lanes share, take now (1 where in range)
  __device__ __forceinline__ float lower(float top) {
    top = other_max(top);
    if (!(top >= 2.f)) return 1.f;
    const float fall = (float)(__builtin_amdgcn_frexp_expf(top) + 6);
    up -= fall;
    return power(-fall);
  }
};
// nonzero: one of 16 packed values is 2 or more (bit 14 of fp16, its highest exponent bit; Inf and NaN have it too)
template <typename X8>
__device__ __forceinline__ unsigned two_or_more(const X8& a, const X8& b) {
  const u32x4 x = __builtin_bit_cast(u32x4, a), y = __builtin_bit_cast(u32x4, b);
  return (x[0] | x[1] | x[2] | x[3] | y[0] | y[1] | y[2] | y[3]) & 0x40004000u;
}
__device__ __forceinline__ float largest(const f32x16& x, float top) {
#pragma unroll
  for (int i = 0; i < 16; i += 2) top = fmaxf(fmaxf(top, fabsf(x[i])), fabsf(x[i + 1]));
  return top;
}

// index of register i of a 32 x 32 result along its rows
__device__ __forceinline__ int reg_row(int i, int half) { return 8 * (i >> 2) + 4 * half + (i & 3); }

// ROWS rows of DP values from global memory into registers and on into an LDS tile.  A thread's place in the tile does not change from tile to
// tile: `at` (bytes from the tile's first row; one add per tile is left, of a uniform pointer) and `to` (LDS) are computed once, and its N
// vectors lie a fixed number of rows apart.  Rows from `valid` on, chunks from D on and rows whose bit is
// set in `skip` (blocked for every query: whatever such a state holds never meets a product) become zeros.
template <typename T, int DP, int ROWS>
struct Stage {
  static constexpr int N = ROWS * (DP / 8) / 256, STEP = 256 / (DP / 8);
  u32x4 r[N];
  unsigned at;
  int row, to;
  bool chunk;
  __device__ __forceinline__ void place(long long stride, int D) {
    const int c = threadIdx.x % (DP / 8);
    row = threadIdx.x / (DP / 8);
    at = (unsigned)(row * (int)stride + c * 8) * 2u;
    to = Tile<DP>::at(row, c);
    chunk = c * 8 < D;
  }
  // tile: address of the tile's first row; step: bytes of STEP rows; valid: rows the tile has; whole: all of it is loaded
  __device__ __forceinline__ void load(const char* tile, long long step, int valid, bool whole, const unsigned* skip, int row0) {
    if (whole) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = *reinterpret_cast<const u32x4*>(tile + i * step + at);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int x = row + STEP * i;
        bool on = chunk && x < valid;
        if (skip && on) on = !((skip[(row0 + x) >> 5] >> ((row0 + x) & 31)) & 1);
        r[i] = u32x4{0u, 0u, 0u, 0u};
        if (on) r[i] = *reinterpret_cast<const u32x4*>(tile + i * step + at);
      }
    }
  }
  __device__ __forceinline__ void store(T* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<u32x4*>(tile + to + i * STEP * Tile<DP>::PITCH) = r[i];
  }
};

// rows of packed query heads -> addresses
struct Row {
  int n, h;
  __device__ Row(const Args& A, int hk, int r) { n = A.G == 1 ? r : (int)((unsigned)r / (unsigned)A.G), h = hk * A.G + (r - n * A.G); }
  __device__ long long packed(const Args& A, int b) const { return (((long long)b * A.Lq + n) * A.Hq + h) * A.D; }
};

// this lane's row (lane & 31) as an operand: DP / 16 steps
template <typename T, int DP>
__device__ __forceinline__ void row_operand(const T* p, int D, bool on, typename Type<T>::x8 (&f)[DP / 16]) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    u32x4 z = {0u, 0u, 0u, 0u};
    if (on && 16 * s + 8 * half < D) z = *reinterpret_cast<const u32x4*>(p + 16 * s + 8 * half);
    f[s] = __builtin_bit_cast(typename Type<T>::x8, z);
  }
}

// 32 dimensions (d0 ..) of this lane's row, times f: the two halves of a wave hold alternate quads of a row, so each hands the other one of every two
// and both write 16 bytes
template <typename T>
__device__ __forceinline__ void put_row(T* row, const f32x16& x, float f, int d0, int D, int half) {
#pragma unroll
  for (int i = 0; i < 16; i += 8) {
    typename Type<T>::x4 a, b;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = (T)(x[i + j] * f), b[j] = (T)(x[i + 4 + j] * f);
    const uint2 ua = __builtin_bit_cast(uint2, a), ub = __builtin_bit_cast(uint2, b);
    const auto lo = __builtin_amdgcn_permlane32_swap(ua.x, ub.x, false, false), hi = __builtin_amdgcn_permlane32_swap(ua.y, ub.y, false, false);
    const int d = d0 + 2 * i + 8 * half;
    if (d < D) *reinterpret_cast<u32x4*>(row + d) = u32x4{lo[0], hi[0], lo[1], hi[1]};
  }
}

// scores of keys key0 .. key0 + 31 against this lane's row: length and mask word
__device__ __forceinline__ void mask_scores(f32x16& s, int key0, int len, bool masked, unsigned word, int half) {
  if (key0 + 32 > len) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (key0 + reg_row(i, half) >= len) s[i] = -kInf;
  }
  if (masked) {
    const unsigned w = word >> (4 * half);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (w & (1u << (8 * (i >> 2) + (i & 3)))) s[i] = -kInf;
  }
}

// a row's mask words of one tile (N blocks of 32 keys from key0 on), read a tile ahead of their use
template <int N>
struct Words {
  unsigned w[N];
  __device__ __forceinline__ void load(const unsigned* words, int key0, int len) {
    if (!words) return;
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = key0 + 32 * i < len ? words[(key0 >> 5) + i] : 0xffffffffu;
  }
};

struct Range { int lo, hi; };
// the keys of split `s`: whole tiles of the sample's own length
__device__ __forceinline__ Range split_range(int len, int splits, int s, int tile) {
  const int tiles = (len + tile - 1) / tile, per = (tiles + splits - 1) / splits;
  return {min(len, s * per * tile), min(len, (s + 1) * per * tile)};
}

// ---- forward ------------------------------------------------------------------------------------------------------------------

// few rows, in blocks of 32: the four waves hold the same rows and share the keys of a tile, 32 each.  Bound by the read of K and V: 16 x 8 x 16384
// keys of 128 (1.07 GB) 198 us = 5.4 TB/s, ragged lengths 153; a single round of workgroups (4 x 8 x 784 of 32) 9 us, which are latency.
template <int DP>
struct Few {
  static constexpr int KW = 4, KT = 32 * KW, TILE = KT * Tile<DP>::PITCH;
  static constexpr int LDS = 2 * TILE * 2 + 2 * KW * 32 * 4;
  static_assert(KW * 32 * DP * 4 <= 2 * TILE * 2, "the join of the waves fits the tiles");
};

__device__ __forceinline__ f32x16 zero16() {
  f32x16 x;
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = 0.f;
  return x;
}

// running softmax of one row block: raw maximum m (of the scores before scaling), sum l of this lane's keys
struct Running {
  float m = -kInf, l = 0.f;
  __device__ __forceinline__ float base(float c) const { return m == -kInf ? 0.f : m * c; }
};

template <typename T, int DP>
__global__ void __launch_bounds__(256, 2) cross_few_kernel(const Args A) {
  typedef Few<DP> F;
  typedef typename Type<T>::x8 x8;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* Kt = reinterpret_cast<T*>(lds);
  T* Vt = Kt + F::TILE;
  const int lane = threadIdx.x & 63, kw = threadIdx.x >> 6, half = lane >> 5, c = lane & 31;
  int id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int r = id % A.tiles * 32 + c;
  id /= A.tiles;
  const int split = id % A.splits;
  id /= A.splits;
  const int hk = id % A.Hk, b = id / A.Hk, len = length_of(A, b);
  const Row row(A, hk, min(r, A.rows - 1));
  const Range keys = split_range(len, A.splits, split, F::KT);
  const char* k = A.k + 2 * (b * A.kb + hk * A.kh);
  const char* v = A.v + 2 * (b * A.vb + hk * A.vh);
  const unsigned* words = A.bits ? A.bits + b * A.mb + row.h * A.mh + row.n * A.mn : nullptr;
  const unsigned* skip = A.bits && A.mn == 0 && (A.mh == 0 || A.G == 1) ? A.bits + b * A.mb + hk * A.mh : nullptr;
  x8 q[DP / 16];
  row_operand<T, DP>(reinterpret_cast<const T*>(A.q) + b * A.qb + row.n * A.qn + row.h * A.qh, A.D, r < A.rows, q);
  f32x16 acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) acc[d] = zero16();
  Running run;
  Stage<T, DP, F::KT> sk, sv;
  sk.place(A.kn, A.D);
  sv.place(A.vn, A.D);
  const bool all = A.D == DP && !skip;
  auto fetch = [&](int k0) {
    const bool whole = all && k0 + F::KT <= len;
    sk.load(k + 2 * k0 * A.kn, 2 * sk.STEP * A.kn, len - k0, whole, skip, k0);
    sv.load(v + 2 * k0 * A.vn, 2 * sv.STEP * A.vn, len - k0, whole, skip, k0);
  };
  Words<1> now = {}, ahead = {};
  if (keys.lo < keys.hi) {
    fetch(keys.lo);
    ahead.load(words, keys.lo + 32 * kw, len);
  }
  for (int k0 = keys.lo; k0 < keys.hi; k0 += F::KT) {
    __syncthreads();
    sk.store(Kt);
    sv.store(Vt);
    now = ahead;
    if (k0 + F::KT < keys.hi) {  // the next tile travels while this one is multiplied
      fetch(k0 + F::KT);
      ahead.load(words, k0 + F::KT + 32 * kw, len);
    }
    __syncthreads();
    f32x16 s;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) s = Type<T>::mfma(operand<T, DP>(Kt, 32 * kw, d), q[d], d ? s : zero16());
    if (A.bits || k0 + F::KT > len) mask_scores(s, k0 + 32 * kw, len, A.bits, now.w[0], half);
    float top = run.m;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[i]);
    top = other_max(top);
    if (__any((top - run.m) * A.c > 8.f)) {  // as in cross_wide_kernel
      const float to = top == -kInf ? 0.f : top * A.c;
      const float alpha = __builtin_amdgcn_exp2f(run.m * A.c - to);
      run.m = top;
      run.l *= alpha;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] *= alpha;
    }
    const float base = run.base(A.c);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], A.c, -base));
      run.l += s[i];
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      // p in two pieces, a product each, and o is as exact as its own rounding (1.0 of that error, 1.2 to 1.4 in one piece): where the keys' read
      // is what takes the time it costs nothing (16 x 8 x 4 rows over 16384 keys of 128: 195 and 196 us), else up to a tenth (15.8 and 17.4)
      const x8 p = pack<T>(s, st), rest = left_off<T>(s, st, p);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        const x8 values_t = operand_t<T, DP>(Vt, 32 * kw + 16 * st, 32 * d);
        acc[d] = Type<T>::mfma(values_t, p, acc[d]);
        acc[d] = Type<T>::mfma(values_t, rest, acc[d]);
      }
    }
  }
  // the waves hold the same rows: join their maxima, sums and results
  const float l = both_sum(run.l), m = run.m;
  float* ml = reinterpret_cast<float*>(lds + 2 * F::TILE * 2);
  float* part = reinterpret_cast<float*>(lds);  // [KW][DP][32]
  __syncthreads();
  if (half == 0) {
    ml[kw * 32 + lane] = m;
    ml[(F::KW + kw) * 32 + lane] = l;
  }
  __syncthreads();
  float top = -kInf, sum = 0.f;
#pragma unroll
  for (int w = 0; w < F::KW; ++w) top = fmaxf(top, ml[w * 32 + c]);
  const float base = top == -kInf ? 0.f : top * A.c;
#pragma unroll
  for (int w = 0; w < F::KW; ++w) sum += ml[(F::KW + w) * 32 + c] * __builtin_amdgcn_exp2f(ml[w * 32 + c] * A.c - base);
  const float f = sum > 0.f ? __builtin_amdgcn_exp2f(m * A.c - base) / sum : (sum == 0.f ? 0.f : sum);
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) part[(kw * DP + 32 * d + reg_row(i, half)) * 32 + c] = acc[d][i] * f;
  __syncthreads();
  if (r >= A.rows) return;
  const long long at = ((long long)b * A.Hk + hk) * A.rows + r, total = (long long)A.B * A.Hk * A.rows;
  // wave w gathers its share of the dimensions
#pragma unroll
  for (int i = 0; i < DP / 8; i += 4) {
    const int d = (kw * 2 + half) * (DP / 8) + i;
    if (d >= A.D) continue;
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = 0.f;
#pragma unroll
      for (int w = 0; w < F::KW; ++w) x[j] += part[(w * DP + d + j) * 32 + c];
    }
    if (A.splits > 1) {
      *reinterpret_cast<float4*>(A.part + (split * total + at) * A.D + d) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
      typename Type<T>::x4 y;
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = (T)x[j];
      *reinterpret_cast<typename Type<T>::x4*>(static_cast<T*>(A.out) + row.packed(A, b) + d) = y;
    }
  }
  if (kw == 0 && half == 0) {
    const float lse = sum > 0.f ? base + log2f(sum) : (sum == 0.f ? -kInf : sum);
    if (A.splits > 1) A.part_lse[split * total + at] = lse;
    else if (A.lse) A.lse[at] = lse == -kInf ? kInf : lse;  // (+inf: the backward pass finds p = 0)
  }
}

// many rows: a wave owns 32, the workgroup 128.  A wave's matrix instructions and its softmax would take turns (a score costs ~5 vector
// instructions of 4 cycles for D / 8 cycles of the matrix pipe), so three tiles are in work at once: while the vector unit turns the scores of
// tile t into probabilities, the matrix pipe forms the scores of tile t + 1 and adds the product of tile t - 1, all in one basic block, where the
// compiler mixes them.  K and V have two LDS buffers each and one barrier a tile: K runs one tile ahead, V one behind.  The loads stand at the head
// of a step (at its end: 720 us instead of 600).
// Bound by the matrix and vector instructions together and, with both at work, by the power that lowers the clock to 1.9 to 2.1 of 2.4 GHz
// (GRBM_GUI_ACTIVE over the kernel's time): 64 x 4096 x 4096 x 128 611 us = 900 TFLOP/s (one tile at a time: 997), 32 x 4099 x 15680 x 64 790 to 810 us
// in a row of calls = 660 TFLOP/s and 850 to 890 after a pause or alone under a profiler (at 64 dimensions a score's exponential weighs twice as much;
// without it 6 % less, without operand reads from LDS 18 %).  Tried without gain: 64 rows a wave (spills), more waves of smaller tiles, loads
// two tiles ahead, no running maximum, chains of maxima and sums.
template <int DP>
struct Wide {
  static constexpr int KB = DP == 128 ? 1 : 2, KT = 32 * KB, RT = 128, TILE = KT * Tile<DP>::PITCH;
  static constexpr int LDS = 4 * TILE * 2;
};

template <typename T, int DP>
__global__ void __launch_bounds__(256, 2) cross_wide_kernel(const Args A) {
  typedef Wide<DP> F;
  typedef typename Type<T>::x8 x8;
  constexpr int KB = F::KB;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* kbuf = reinterpret_cast<T*>(lds);
  T* vbuf = kbuf + 2 * F::TILE;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  int id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int tile = id % A.tiles;
  id /= A.tiles;
  const int split = id % A.splits;
  id /= A.splits;
  const int hk = id % A.Hk, b = id / A.Hk;
  const int r = tile * F::RT + wave * 32 + (lane & 31), len = length_of(A, b);
  const Range keys = split_range(len, A.splits, split, F::KT);
  const char* k = A.k + 2 * (b * A.kb + hk * A.kh);
  const char* v = A.v + 2 * (b * A.vb + hk * A.vh);
  const unsigned* skip = A.bits && A.mn == 0 && (A.mh == 0 || A.G == 1) ? A.bits + b * A.mb + hk * A.mh : nullptr;
  const unsigned* words = nullptr;
  x8 q[DP / 16];
  {
    const Row row(A, hk, min(r, A.rows - 1));
    row_operand<T, DP>(reinterpret_cast<const T*>(A.q) + b * A.qb + row.n * A.qn + row.h * A.qh, A.D, r < A.rows, q);
    if (A.bits) words = A.bits + b * A.mb + row.h * A.mh + row.n * A.mn;
  }
  f32x16 acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) acc[d] = zero16();
  Stage<T, DP, F::KT> sk, sv;
  sk.place(A.kn, A.D);
  sv.place(A.vn, A.D);
  const bool all = A.D == DP && !skip;
  const int steps = (keys.hi - keys.lo + F::KT - 1) / F::KT;
  auto fetch_k = [&](Stage<T, DP, F::KT>& to, int t) {
    const int k0 = keys.lo + t * F::KT;
    to.load(k + 2 * k0 * A.kn, 2 * sk.STEP * A.kn, len - k0, all && k0 + F::KT <= len, skip, k0);
  };
  auto fetch_v = [&](int t) {
    const int k0 = keys.lo + t * F::KT;
    sv.load(v + 2 * k0 * A.vn, 2 * sv.STEP * A.vn, len - k0, all && k0 + F::KT <= len, skip, k0);
  };
  x8 p[KB][2];  // the probabilities of the tile before, in the order of the second product
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) p[kb][0] = p[kb][1] = pack<T>(zero16(), 0);
  auto scores = [&](const T* Kt, f32x16 (&x)[KB]) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) x[kb] = Type<T>::mfma(operand<T, DP>(Kt, kb * 32, d), q[d], d ? x[kb] : zero16());
  };
  auto add_values = [&](const T* Vt) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] = Type<T>::mfma(operand_t<T, DP>(Vt, kb * 32 + 16 * st, 32 * d), p[kb][st], acc[d]);
  };
  Running run;
  // tile t: its scores s; the scores of tile t + 1 go to `next`; `now`, `other`: the buffers of tile t and of its neighbours
  Words<KB> mask = {};
  auto step = [&](int t, f32x16 (&s)[KB], f32x16 (&next)[KB], int now, int other) {
    const int k0 = keys.lo + t * F::KT;
    if (t + 2 < steps) fetch_k(sk, t + 2);
    fetch_v(t);
    __syncthreads();
    if (A.bits || k0 + F::KT > len) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) mask_scores(s[kb], k0 + 32 * kb, len, A.bits, mask.w[kb], half);
      mask.load(words, k0 + F::KT, len);
    }
    float top = run.m;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kb][i]);
    top = other_max(top);
    // the reference point only moves once a score passes it by 2^8 in the result: p then stays under 2^8, in the range of every type, and
    // the accumulators are rescaled a few times in all instead of once a tile
    if (__any((top - run.m) * A.c > 8.f)) {  // (-inf against -inf: NaN, no)
      add_values(vbuf + other);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) p[kb][0] = p[kb][1] = pack<T>(zero16(), 0);
      const float to = top == -kInf ? 0.f : top * A.c;
      const float alpha = __builtin_amdgcn_exp2f(run.m * A.c - to);  // (m = -inf: 0)
      run.m = top;
      run.l *= alpha;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] *= alpha;
    }
    const float base = run.base(A.c);
    scores(kbuf + other, next);  // (behind the last tile: what lies in the buffer, not used)
    add_values(vbuf + other);
    // p is rounded to the tensor's type for the product (half a step relative to each p); its sum l keeps 32 bits
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[kb][i] = __builtin_amdgcn_exp2f(fmaf(s[kb][i], A.c, -base));
        run.l += s[kb][i];
      }
      p[kb][0] = pack<T>(s[kb], 0);
      p[kb][1] = pack<T>(s[kb], 1);
    }
    sk.store(kbuf + now);  // (no tile t + 2: what was there, not used)
    sv.store(vbuf + now);
  };
  if (steps > 0) {
    Stage<T, DP, F::KT> k1 = sk;
    fetch_k(sk, 0);
    if (steps > 1) fetch_k(k1, 1);
    mask.load(words, keys.lo, len);
    sk.store(kbuf);
    if (steps > 1) k1.store(kbuf + F::TILE);
    for (int i = threadIdx.x; i < F::TILE / 8; i += 256) reinterpret_cast<u32x4*>(vbuf + F::TILE)[i] = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
    f32x16 s0[KB], s1[KB];
    scores(kbuf, s0);
    for (int t = 0;; t += 2) {
      step(t, s0, s1, 0, F::TILE);
      if (t + 1 >= steps) break;
      step(t + 1, s1, s0, F::TILE, 0);
      if (t + 2 >= steps) break;
    }
    __syncthreads();
    add_values(vbuf + ((steps - 1) & 1) * F::TILE);
  }
  const float l = both_sum(run.l);
  if (r >= A.rows) return;
  const Row row(A, hk, r);
  const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  const long long at = ((long long)b * A.Hk + hk) * A.rows + r;
  if (A.splits > 1) {
    float* o = A.part + (split * ((long long)A.B * A.Hk * A.rows) + at) * A.D;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int dd = 32 * d + reg_row(i, half);
        if (dd < A.D) *reinterpret_cast<float4*>(o + dd) = make_float4(acc[d][i] * f, acc[d][i + 1] * f, acc[d][i + 2] * f, acc[d][i + 3] * f);
      }
  } else {
    T* o = static_cast<T*>(A.out) + row.packed(A, b);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) put_row(o, acc[d], f, 32 * d, A.D, half);
  }
  if (half == 0) {
    const float lse = l > 0.f ? run.base(A.c) + log2f(l) : (l == 0.f ? -kInf : l);
    if (A.splits > 1) A.part_lse[split * ((long long)A.B * A.Hk * A.rows) + at] = lse;
    else if (A.lse) A.lse[at] = lse == -kInf ? kInf : lse;  // (+inf: the backward pass finds p = 0)
  }
}

// ---- backward -----------------------------------------------------------------------------------------------------------------

// o . do of this lane's row as the diagonal of a product: the same order of summation as do . v, so a row that sees one key has ds = 0 exactly
template <typename T, int DP>
__device__ __forceinline__ float row_dot(const typename Type<T>::x8 (&o)[DP / 16], const typename Type<T>::x8 (&g)[DP / 16]) {
  f32x16 x = zero16();
#pragma unroll
  for (int d = 0; d < DP / 16; ++d) x = Type<T>::mfma(o[d], g[d], x);
  const int c = threadIdx.x & 31;
  float delta = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (4 * (c >> 3) + (c & 3) == i) delta = x[i];
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(delta), __float_as_uint(delta), false, false);
  return __uint_as_float((c >> 2) & 1 ? sw[1] : sw[0]);
}

// dq: the walk over the keys again, p from the saved lse; per tile two score-sized products and the one with K.  The scores of tile t + 1 are
// formed in the same basic block in which the vector unit turns those of tile t into ds, so there are three buffers (t, t + 1, and t + 2 filling).
// 64 x 4096 x 4096 x 128: 750 to 800 us = 1.05 PFLOP/s (6 S D), like the forward pass at its power limit (tiles one at a time: 1395; loads at the
// step's end: 815).
// RW = 4: a wave owns 32 rows; RW = 1 (blocks of 32 rows): the waves share the keys of a tile.
template <int DP, int RW>
struct Dq {
  static constexpr int KW = 4 / RW, KB = RW == 4 && DP < 128 ? 2 : 1, KT = 32 * KB * KW, RT = 32 * RW, TILE = KT * Tile<DP>::PITCH;
  static constexpr int BUFS = RW == 4 ? 3 : 1, TILES = 2 * BUFS * TILE * 2, LDS = TILES + (KW > 1 ? KW * 32 * 4 : 0);
  static_assert(KW == 1 || KW * 32 * DP * 4 <= 2 * TILE * 2, "the join of the waves fits the tiles");
};

template <typename T, int DP, int RW>
__global__ void __launch_bounds__(256, RW == 1 && DP == 128 ? 1 : 2) cross_dq_kernel(const Args A) {
  typedef Dq<DP, RW> F;
  typedef typename Type<T>::x8 x8;
  constexpr int KB = F::KB;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* kbuf = reinterpret_cast<T*>(lds);
  T* vbuf = kbuf + F::BUFS * F::TILE;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int rw = wave % RW, kw = wave / RW;
  int id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int tile = id % A.tiles;
  id /= A.tiles;
  const int split = id % A.splits;
  id /= A.splits;
  const int hk = id % A.Hk, b = id / A.Hk;
  const int r = tile * F::RT + rw * 32 + (lane & 31), len = length_of(A, b);
  const bool on = r < A.rows;
  const Range keys = split_range(len, A.splits, split, F::KT);
  const char* k = A.k + 2 * (b * A.kb + hk * A.kh);
  const char* v = A.v + 2 * (b * A.vb + hk * A.vh);
  const unsigned* skip = A.bits && A.mn == 0 && (A.mh == 0 || A.G == 1) ? A.bits + b * A.mb + hk * A.mh : nullptr;
  const unsigned* words = nullptr;
  const long long at = ((long long)b * A.Hk + hk) * A.rows + r;
  Stage<T, DP, F::KT> sk, sv;
  sk.place(A.kn, A.D);
  sv.place(A.vn, A.D);
  const bool all = A.D == DP && !skip;
  auto fetch = [&](Stage<T, DP, F::KT>& sk, Stage<T, DP, F::KT>& sv, int k0) {
    const bool whole = all && k0 + F::KT <= len;
    sk.load(k + 2 * k0 * A.kn, 2 * sk.STEP * A.kn, len - k0, whole, skip, k0);
    sv.load(v + 2 * k0 * A.vn, 2 * sv.STEP * A.vn, len - k0, whole, skip, k0);
  };
  const int steps = (keys.hi - keys.lo + F::KT - 1) / F::KT;
  // the first tiles travel together with the rows
  Stage<T, DP, F::KT> k1 = sk, v1 = sv;
  if (steps > 0) fetch(sk, sv, keys.lo);
  if (RW == 4 && steps > 1) fetch(k1, v1, keys.lo + F::KT);
  x8 q[DP / 16], g[DP / 16];
  float delta = 0.f;
  {
    const Row row(A, hk, min(r, A.rows - 1));
    const long long here = row.packed(A, b);
    if (A.bits) words = A.bits + b * A.mb + row.h * A.mh + row.n * A.mn;
    row_operand<T, DP>(reinterpret_cast<const T*>(A.q) + b * A.qb + row.n * A.qn + row.h * A.qh, A.D, on, q);
    row_operand<T, DP>(static_cast<const T*>(A.dout) + here, A.D, on, g);
    x8 o[DP / 16];
    row_operand<T, DP>(static_cast<const T*>(A.o) + here, A.D, on, o);
    delta = row_dot<T, DP>(o, g);
  }
  const float lse = on ? A.lse[at] : kInf;
  f32x16 acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) acc[d] = zero16();
  auto scores = [&](const T* Kt, f32x16 (&s)[KB]) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) s[kb] = Type<T>::mfma(operand<T, DP>(Kt, (kw * KB + kb) * 32, d), q[d], d ? s[kb] : zero16());
  };
  Words<KB> bits = {};
  auto mask = [&](int k0, f32x16 (&s)[KB]) {
    if (A.bits || k0 + F::KT > len) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) mask_scores(s[kb], k0 + (kw * KB + kb) * 32, len, A.bits, bits.w[kb], half);
      bits.load(words, k0 + F::KT + kw * KB * 32, len);
    }
  };
  // ds, rounded to the tensor's type for the product (half a step relative to each).  States that no query sees were staged as zeros, so dp is
  // finite where p is zero by a length or a shared mask.  In blocks of 32 rows and up to 32 dimensions, where a product costs little, what the
  // rounding left off follows in a product of its own: dq came out 1.45 to 1.55 times the error of its own rounding, most of it at 16 dimensions,
  // and is now at 1.05 (40 x 8 x 100 rows over 784 keys of 32: 28 -> 33 us, 16 x 8 x 4 rows over 16384 of 128: 188 -> 196).
  constexpr int PIECES = DP == 32 || RW == 1 ? 2 : 1;
  typedef x8 Grad[KB][2][PIECES];
  constexpr bool kHeld = std::is_same_v<T, _Float16>;
  Held hold;
  float base = kHeld ? lse - hold.up : lse;  // (p comes at 2^up)
  auto gradient = [&](const T* Vt, const f32x16 (&s)[KB], f32x16 (&x)[KB]) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      f32x16 dp;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) dp = Type<T>::mfma(operand<T, DP>(Vt, (kw * KB + kb) * 32, d), g[d], d ? dp : zero16());
#pragma unroll
      for (int i = 0; i < 16; ++i) x[kb][i] = __builtin_amdgcn_exp2f(fmaf(s[kb][i], A.c, -base));
#pragma unroll
      for (int i = 0; i < 16; ++i) x[kb][i] *= dp[i] - delta;
    }
  };
  auto round_off = [&](f32x16 (&x)[KB], Grad& ds) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int st = 0; st < 2; ++st) ds[kb][st][0] = pack<T>(x[kb], st);
    if constexpr (kHeld) {
      unsigned large = 0u;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) large |= two_or_more(ds[kb][0][0], ds[kb][1][0]);
      if (__any(large)) {
        float top = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) top = largest(x[kb], top);
        const float f = hold.lower(top);
        base = lse - hold.up;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i) x[kb][i] *= f;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[d][i] *= f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int st = 0; st < 2; ++st) ds[kb][st][0] = pack<T>(x[kb], st);
      }
    }
    if constexpr (PIECES == 2) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int st = 0; st < 2; ++st) ds[kb][st][1] = left_off<T>(x[kb], st, ds[kb][st][0]);
    }
  };
  // Delta = o . do carries the rounding of o and of the probabilities that made it, and over few keys that is as large as the rounding of ds.
  // Where this workgroup has the whole row in LDS, delta + sum_j p_j (dp_j - delta) takes its place: the same number without the roundings
  // (16 keys: dq and dk 1.56 -> 1.42 times the error of one rounding; 60 of which a mask leaves 24: 1.51 -> 1.42; longer walks have 1.43 to 1.47
  // without it).  It costs a second look at those tiles: 4 x 10 x 4096 rows against 77 keys 29 -> 35 us.
  const bool at_hand = keys.lo == 0 && keys.hi == len && steps <= F::BUFS;
  auto missing = [&](const T* Kt, const T* Vt, int k0) {
    f32x16 s[KB];
    scores(Kt, s);
    mask(k0, s);
    float sum = 0.f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      f32x16 dp;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) dp = Type<T>::mfma(operand<T, DP>(Vt, (kw * KB + kb) * 32, d), g[d], d ? dp : zero16());
#pragma unroll
      for (int i = 0; i < 16; ++i) sum += __builtin_amdgcn_exp2f(fmaf(s[kb][i], A.c, -lse)) * (dp[i] - delta);
    }
    bits.load(words, keys.lo + kw * KB * 32, len);
    return both_sum(sum);
  };
  auto add_keys = [&](const T* Kt, const Grad& ds) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          const x8 keys_t = operand_t<T, DP>(Kt, (kw * KB + kb) * 32 + 16 * st, 32 * d);
#pragma unroll
          for (int i = 0; i < PIECES; ++i) acc[d] = Type<T>::mfma(keys_t, ds[kb][st][i], acc[d]);
        }
  };
  bits.load(words, keys.lo + kw * KB * 32, len);
  if (RW == 1) {
    for (int t = 0; t < steps; ++t) {
      const int k0 = keys.lo + t * F::KT;
      __syncthreads();
      sk.store(kbuf);
      sv.store(vbuf);
      if (t + 1 < steps) fetch(sk, sv, k0 + F::KT);
      __syncthreads();
      if (at_hand) {
        float* sums = reinterpret_cast<float*>(lds + F::TILES);
        const float sum = missing(kbuf, vbuf, k0);
        if (half == 0) sums[wave * 32 + lane] = sum;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < F::KW; ++w) delta += sums[w * 32 + (lane & 31)];
      }
      f32x16 s[KB], x[KB];
      Grad ds;
      scores(kbuf, s);
      mask(k0, s);
      gradient(vbuf, s, x);
      round_off(x, ds);
      add_keys(kbuf, ds);
    }
  } else if (steps > 0) {
    sk.store(kbuf);
    sv.store(vbuf);
    if (steps > 1) {
      k1.store(kbuf + F::TILE);
      v1.store(vbuf + F::TILE);
    }
    if (at_hand && steps == 3) {
      fetch(sk, sv, keys.lo + 2 * F::KT);
      sk.store(kbuf + 2 * F::TILE);
      sv.store(vbuf + 2 * F::TILE);
    }
    __syncthreads();
    if (at_hand) {
      float sum = 0.f;
      for (int t = 0; t < steps; ++t) {
        if (t) bits.load(words, keys.lo + t * F::KT, len);
        sum += missing(kbuf + t * F::TILE, vbuf + t * F::TILE, keys.lo + t * F::KT);
      }
      delta += sum;
    }
    f32x16 s[KB];
    scores(kbuf, s);
    int kt = 0, kn = F::TILE, kf = 2 * F::TILE;  // K (and V) of tile t, t + 1, t + 2
    for (int t = 0; t < steps; ++t) {
      const int k0 = keys.lo + t * F::KT;
      if (t + 2 < steps) fetch(sk, sv, k0 + 2 * F::KT);
      __syncthreads();
      mask(k0, s);
      f32x16 x[KB];
      Grad ds;
      gradient(vbuf + kt, s, x);
      if constexpr (kHeld) scores(kbuf + kn, s);  // (ahead of the branch in round_off, so that they share a basic block with the gradient)
      round_off(x, ds);
      if constexpr (!kHeld) scores(kbuf + kn, s);  // (behind the last tile: what lies in the buffer, not used)
      add_keys(kbuf + kt, ds);
      sk.store(kbuf + kf);  // tile t + 2 (none left: what was there, not used)
      sv.store(vbuf + kf);
      const int y = kt;
      kt = kn, kn = kf, kf = y;
    }
  }
  if constexpr (kHeld) {
    const float back = Held::power(-hold.up);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] *= back;
  }
  if (on && half == 0 && kw == 0 && split == 0) A.delta[at] = delta;
  auto store = [&](int d, const float (&x)[4]) {
    if (d >= A.D) return;
    if (A.splits > 1) {
      float* o = A.part + (split * ((long long)A.B * A.Hk * A.rows) + at) * A.D + d;
      *reinterpret_cast<float4*>(o) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
      typename Type<T>::x4 y;
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = (T)(x[j] * A.scale);
      const Row row(A, hk, r);
      *reinterpret_cast<typename Type<T>::x4*>(static_cast<T*>(A.out) + row.packed(A, b) + d) = y;
    }
  };
  if constexpr (F::KW > 1) {
    float* part = reinterpret_cast<float*>(lds);
    __syncthreads();
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) part[(kw * DP + 32 * d + reg_row(i, half)) * 32 + (lane & 31)] = acc[d][i];
    __syncthreads();
    if (!on) return;
#pragma unroll
    for (int i = 0; i < DP / 8; i += 4) {
      const int d = (kw * 2 + half) * (DP / 8) + i;
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = 0.f;
#pragma unroll
        for (int w = 0; w < F::KW; ++w) x[j] += part[(w * DP + d + j) * 32 + (lane & 31)];
      }
      store(d, x);
    }
  } else {
    if (!on) return;
    if (A.splits > 1) {
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float x[4] = {acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]};
          store(32 * d + reg_row(i, half), x);
        }
    } else {
      T* o = static_cast<T*>(A.out) + Row(A, hk, r).packed(A, b);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) put_row(o, acc[d], A.scale, 32 * d, A.D, half);
    }
  }
}

// dk, dv: a wave owns 32 keys, the workgroup walks the rows of all G heads.  Score tiles are rows x keys here (a lane owns a key), so they are
// the B operands of dV^T = dO^T P and dK^T = Q^T dS; lse and delta of a tile's rows lie in LDS.  Tiles of 32 rows: of 64, at 32 dimensions, they took
// all 256 registers and 40 x 8 x 100 rows and 784 keys 35.6 us instead of 30.7 (4 x 8 x 2000 and 2000 keys, enough work a wave: 60.8 and 65.0).
template <typename T, int DP>
struct Bwd {
  static constexpr int KT = 128, RT = 32;
  static constexpr int TILE = 2 * RT * Tile<DP>::PITCH * 2, SIDE = 2 * RT * 4 + 4 * RT * 4;  // Q and dO; lse, delta and the four waves' mask words
  static constexpr int BUF = TILE + SIDE, LDS = 3 * BUF;
};

template <typename T, int DP>
__global__ void __launch_bounds__(256, DP == 128 ? 1 : 2) cross_dkv_kernel(const Args A) {
  typedef Bwd<T, DP> F;
  typedef typename Type<T>::x8 x8;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  int id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int tile = id % A.tiles;
  id /= A.tiles;
  const int split = id % A.splits;
  id /= A.splits;
  const int hk = id % A.Hk, b = id / A.Hk;
  const int len = length_of(A, b), key0 = tile * F::KT + wave * 32, key = key0 + (lane & 31);
  const unsigned* skip = A.bits && A.mn == 0 && (A.mh == 0 || A.G == 1) ? A.bits + b * A.mb + hk * A.mh : nullptr;
  bool open = key < len;
  if (skip && open) open = !((skip[key >> 5] >> (key & 31)) & 1);
  x8 k[DP / 16], v[DP / 16];
  row_operand<T, DP>(reinterpret_cast<const T*>(A.k) + b * A.kb + hk * A.kh + key * A.kn, A.D, open, k);
  row_operand<T, DP>(reinterpret_cast<const T*>(A.v) + b * A.vb + hk * A.vh + key * A.vn, A.D, open, v);
  f32x16 ak[DP / 32], av[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) ak[d] = av[d] = zero16();
  const int row_tiles = (A.rows + F::RT - 1) / F::RT, per = (row_tiles + A.splits - 1) / A.splits;
  const int lo = split * per, hi = tile * F::KT < len ? min(row_tiles, (split + 1) * per) : lo;
  const T* q = reinterpret_cast<const T*>(A.q) + b * A.qb;
  const T* g = static_cast<const T*>(A.dout);
  const long long side = ((long long)b * A.Hk + hk) * A.rows;
  // fp16 holds p as 2^12 p: over thousands of keys most of p is under 2^-14, where the type runs out of digits (16384 keys: dv 1.55 -> 1.42 times
  // the error of one rounding); p <= 1 stays in range.  So lse comes 12 less and dv ends with the reverse; ds has a scale of its own (Held).
  constexpr bool half_type = std::is_same_v<T, _Float16>;
  constexpr float kDown = half_type ? 1.f / 4096.f : 1.f;
  Held hold;
  float lift = Held::power(hold.up - 12.f);
  // a thread's vectors of a tile, of Q and of dO by turns (one vector: half of the threads each); where G divides a tile's rows they move on by the
  // same distance from tile to tile
  constexpr int N = 2 * F::RT * (DP / 8) / 256, STEP = 256 / (DP / 8);
  const bool even = F::RT % A.G == 0 && A.D == DP;
  const int c = threadIdx.x % (DP / 8), x0 = threadIdx.x / (DP / 8);
  const int to = Tile<DP>::at(x0, c);
  const long long qstep = F::RT / A.G * A.qn, gstep = (long long)(F::RT / A.G) * A.Hq * A.D;
  auto of_q = [&](int i) { return N == 1 ? x0 < F::RT : i % 2 == 0; };
  auto row_of = [&](int i) { return N == 1 ? x0 % F::RT : x0 + STEP * (i / 2); };
  long long at[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const Row row(A, hk, row_of(i));
    at[i] = (of_q(i) ? row.n * A.qn + row.h * A.qh : row.packed(A, b)) + c * 8;
  }
  u32x4 held[N];
  float rl = 0.f;
  unsigned rm = 0u;
  auto fetch = [&](int rt) {
    if (even && (rt + 1) * F::RT <= A.rows) {
#pragma unroll
      for (int i = 0; i < N; ++i) held[i] = *reinterpret_cast<const u32x4*>((of_q(i) ? q + rt * qstep : g + rt * gstep) + at[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = rt * F::RT + row_of(i);
        held[i] = u32x4{0u, 0u, 0u, 0u};
        if (r < A.rows && c * 8 < A.D) {
          const Row row(A, hk, r);
          held[i] = *reinterpret_cast<const u32x4*>(of_q(i) ? q + row.n * A.qn + row.h * A.qh + c * 8 : g + row.packed(A, b) + c * 8);
        }
      }
    }
    if (threadIdx.x < 2 * F::RT) {  // the first RT threads: lse, the next: delta
      const int r = rt * F::RT + threadIdx.x % F::RT;
      const float* from = threadIdx.x < F::RT ? A.lse : A.delta;
      rl = r < A.rows ? from[side + r] : (threadIdx.x < F::RT ? kInf : 0.f);
      if constexpr (half_type) rl = threadIdx.x < F::RT ? rl - 12.f : rl;
    }
    if (A.bits) {
      const int x = threadIdx.x, r = rt * F::RT + x % F::RT, w = tile * 4 + x / F::RT;
      rm = 0xffffffffu;
      if (x < 4 * F::RT && r < A.rows && w * 32 < A.Lk) {
        const Row row(A, hk, r);
        rm = A.bits[b * A.mb + row.h * A.mh + row.n * A.mn + w];
      }
    }
  };
  auto park = [&](char* buf) {
    T* Qt = reinterpret_cast<T*>(buf);
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<u32x4*>(Qt + to + (i / 2 * STEP + i % 2 * F::RT) * Tile<DP>::PITCH) = held[i];
    if (threadIdx.x < 2 * F::RT) reinterpret_cast<float*>(buf + F::TILE)[threadIdx.x] = rl;
    if (A.bits && threadIdx.x < 4 * F::RT) reinterpret_cast<unsigned*>(buf + F::TILE + 2 * F::RT * 4)[threadIdx.x] = rm;
  };
  auto mask = [&](const char* buf, f32x16& s) {
    if (!A.bits) return;
    const unsigned* Mt = reinterpret_cast<const unsigned*>(buf + F::TILE + 2 * F::RT * 4) + wave * F::RT;
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const uint4 w = *reinterpret_cast<const uint4*>(Mt + reg_row(i, half));
      const unsigned w4[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((w4[j] >> (lane & 31)) & 1) s[i + j] = -kInf;
    }
  };
  // The compiler places an LDS read right before the instruction that needs it, and with one or two waves on a SIMD its latency then shows at every
  // product.  So a tile is worked in four stages that nothing is moved across; a stage's products take operands that the stage before has read,
  // and its vector instructions do not wait for its own products (64 x 4096 x 4096 x 128: 1750 us as one block, now 1270 to 1380 = 830 TFLOP/s of
  // 8 S D, one wave a SIMD):
  //     dP of tile t               | p = exp2(S)               | reads Q of tile t + 1
  //     S of tile t + 1            | ds = p (dP - delta)       | reads dO^T of tile t
  //     dV += dO^T p               |                           | reads Q^T of tile t
  //     dK += Q^T ds               |                           | reads dO and lse of tile t + 1
  constexpr int ND = DP / 16, NT = DP / 32;
  typedef x8 Rows[ND];     // operands of a product over the head dimension
  typedef x8 Cols[2][NT];  // operands of a product over the tile's rows
  auto read_rows = [&](const T* Xt, Rows& x) {
#pragma unroll
    for (int d = 0; d < ND; ++d) x[d] = operand<T, DP>(Xt, 0, d);
  };
  auto read_cols = [&](const T* Xt, Cols& x) {
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int d = 0; d < NT; ++d) x[st][d] = operand_t<T, DP>(Xt, 16 * st, 32 * d);
  };
  auto q_tile = [&](int buf) { return reinterpret_cast<const T*>(lds + buf); };
  auto g_tile = [&](int buf) { return reinterpret_cast<const T*>(lds + buf) + F::RT * Tile<DP>::PITCH; };
  auto over_rows = [&](const Rows& x, const x8 (&y)[ND], f32x16& o) {
#pragma unroll
    for (int d = 0; d < ND; ++d) o = Type<T>::mfma(x[d], y[d], d ? o : zero16());
  };
  auto over_cols = [&](const Cols& x, const x8 (&y)[2], f32x16 (&o)[NT]) {
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int d = 0; d < NT; ++d) o[d] = Type<T>::mfma(x[st][d], y[st], o[d]);
  };
  // a value per row (lse or delta) for this lane's 16 rows
  auto read_side = [&](const float* side_, f32x16& x) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const float4 y = *reinterpret_cast<const float4*>(side_ + reg_row(i, half));
      x[i] = y.x, x[i + 1] = y.y, x[i + 2] = y.z, x[i + 3] = y.w;
    }
  };
  auto lse_of = [&](int buf) { return reinterpret_cast<const float*>(lds + buf + F::TILE); };
  // ds to its scale (fp16) and type.  With one wave a SIMD the scale, the check and the branch stand beside the products of dV, where the vector unit is
  // free (64 x 4096 x 4096 x 128: 2180 -> 2030 us; ds without a scale 1910); at 32 dimensions x would live longer than three workgroups a CU
  // have registers for (40 x 8 x 100 rows and 784 keys, the whole pass: 70.5 against 76.7).
  constexpr bool kLate = half_type && DP == 128;
  auto round_off = [&](f32x16& x, x8 (&ds)[2]) {
    if constexpr (half_type) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] *= lift;
    }
    ds[0] = pack<T>(x, 0);
    ds[1] = pack<T>(x, 1);
    if constexpr (half_type) {
      if (__any(two_or_more(ds[0], ds[1]))) {
        const float f = hold.lower(largest(x, 0.f));
        lift *= f;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= f;
#pragma unroll
        for (int d = 0; d < NT; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) ak[d][i] *= f;
        ds[0] = pack<T>(x, 0);
        ds[1] = pack<T>(x, 1);
      }
    }
  };
  if (lo < hi) {
    fetch(lo);
    park(lds);
    if (lo + 1 < hi) {
      fetch(lo + 1);
      park(lds + F::BUF);
    }
    __syncthreads();
    f32x16 s, dp, x, L;
    Rows rows;
    Cols cols, cols2;
    read_rows(q_tile(0), rows);
    over_rows(rows, k, s);
    read_rows(g_tile(0), rows);
    read_side(lse_of(0), L);
    int bt = 0, bn = F::BUF, bf = 2 * F::BUF;  // buffers of tile t, t + 1, t + 2
    for (int rt = lo; rt < hi; ++rt) {
      if (rt + 2 < hi) fetch(rt + 2);
      __syncthreads();
      mask(lds + bt, s);
      over_rows(rows, v, dp);
      Rows next;
      read_rows(q_tile(bn), next);  // (behind the last tile: what lies in the buffer, not used)
      x8 p[2], ds[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = __builtin_amdgcn_exp2f(fmaf(s[i], A.c, -L[i]));
      // p, and ds below, are rounded to the tensor's type for the products (half a step relative to each)
      p[0] = pack<T>(x, 0);
      p[1] = pack<T>(x, 1);
      read_side(lse_of(bt) + F::RT, L);  // delta
      __builtin_amdgcn_sched_barrier(0);
      over_rows(next, k, s);
      read_cols(g_tile(bt), cols);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] *= dp[i] - L[i];
      if constexpr (!kLate) round_off(x, ds);
      __builtin_amdgcn_sched_barrier(0);
      over_cols(cols, p, av);
      read_cols(q_tile(bt), cols2);
      if constexpr (kLate) round_off(x, ds);
      __builtin_amdgcn_sched_barrier(0);
      over_cols(cols2, ds, ak);
      read_rows(g_tile(bn), rows);
      read_side(lse_of(bn), L);
      park(lds + bf);
      const int y = bt;
      bt = bn, bn = bf, bf = y;
    }
  }
  if constexpr (half_type) {
    const float back = Held::power(-hold.up);
#pragma unroll
    for (int d = 0; d < NT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) ak[d][i] *= back;
  }
  if (key >= A.Lk) return;
  if (!open) {  // keys behind the length or blocked for all: zeros
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) ak[d] = av[d] = zero16();
  }
  const long long here = (((long long)b * A.Lk + key) * A.Hk + hk) * A.D, all = (long long)A.B * A.Lk * A.Hk * A.D;
  if (A.splits > 1) {
    float* o = A.part + 2 * split * all + here;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int dd = 32 * d + reg_row(i, half);
        if (dd >= A.D) continue;
        *reinterpret_cast<float4*>(o + dd) = make_float4(ak[d][i] * A.scale, ak[d][i + 1] * A.scale, ak[d][i + 2] * A.scale, ak[d][i + 3] * A.scale);
        *reinterpret_cast<float4*>(o + all + dd) = make_float4(av[d][i] * kDown, av[d][i + 1] * kDown, av[d][i + 2] * kDown, av[d][i + 3] * kDown);
      }
  } else {
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
      put_row(static_cast<T*>(A.dk) + here, ak[d], A.scale, 32 * d, A.D, half);
      put_row(static_cast<T*>(A.dv) + here, av[d], kDown, 32 * d, A.D, half);
    }
  }
}

// ---- the splits of a row joined, 8 values (a vector) at a time ------------------------------------------------------------------
// A load's latency is ~0.65 us, and a thread that walks 64 splits one by one takes 42 us.  So P lanes share the splits of a vector, four loads
// in flight each (the vectors of a wave stay side by side, the lanes of one lie 64 / P apart), and a tree over the lanes ends it: 4.1 us for 64
// splits of 4 x 8 rows, 6.0 for 128, little more than a launch.

__host__ __device__ inline int lanes_of(int splits) {
  int P = 1;
  while (P < 32 && 4 * P < splits) P *= 2;
  return P;
}

struct Share {
  int P, apart, first;  // lanes of a vector, their distance, this lane's first split
  long long vector;
  __device__ explicit Share(int splits) {
    const int lane = threadIdx.x & 63;
    P = lanes_of(splits), apart = 64 / P, first = lane / apart;
    vector = (blockIdx.x * 256ll + threadIdx.x) / 64 * apart + lane % apart;
  }
  // sum of the vectors at from + s * step over the splits s, each times weight(s)
  template <typename F>
  __device__ f32x8 sum(const float* from, long long step, int splits, F weight) const {
    f32x8 x = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s0 = first; s0 < splits; s0 += 4 * P) {
      f32x8 y[4];
      float w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int s = min(s0 + u * P, splits - 1);
        y[u] = *reinterpret_cast<const f32x8*>(from + s * step);
        w[u] = weight(s);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (s0 + u * P < splits) x += y[u] * w[u];
    }
    for (int o = apart; o < 64; o *= 2)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] += __shfl_xor(x[i], o);
    return x;
  }
};

template <typename T>
__global__ void __launch_bounds__(256) cross_join_kernel(const Args A) {
  const int per = A.D / 8;
  const long long total = (long long)A.B * A.Hk * A.rows;
  const Share mine(A.splits);
  const bool on = mine.vector < total * per;
  const long long i = on ? mine.vector : 0, at = fast_div(i, per);
  const int d = (int)(i - at * per) * 8;
  const float* lse = A.part_lse + at;
  float top = -kInf, sum = 0.f;
#pragma unroll 4
  for (int s = mine.first; s < A.splits; s += mine.P) top = fmaxf(top, lse[s * total]);
  for (int o = mine.apart; o < 64; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
  const float base = top == -kInf ? 0.f : top;
#pragma unroll 4
  for (int s = mine.first; s < A.splits; s += mine.P) sum += __builtin_amdgcn_exp2f(lse[s * total] - base);
  for (int o = mine.apart; o < 64; o *= 2) sum += __shfl_xor(sum, o);
  const f32x8 x = mine.sum(A.part + at * A.D + d, total * A.D, A.splits, [&](int s) { return __builtin_amdgcn_exp2f(lse[s * total] - base); });
  if (!on || mine.first) return;
  const float f = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  const long long bh = at / A.rows;
  const Row row(A, (int)(bh % A.Hk), (int)(at % A.rows));
  *reinterpret_cast<typename Type<T>::x8*>(static_cast<T*>(A.out) + row.packed(A, (int)(bh / A.Hk)) + d) =
      __builtin_convertvector(x * f, typename Type<T>::x8);
  if (A.lse && d == 0) A.lse[at] = sum > 0.f ? base + log2f(sum) : (sum == 0.f ? kInf : sum);
}

template <typename T>
__global__ void __launch_bounds__(256) cross_dq_sum_kernel(const Args A) {
  const int per = A.D / 8;
  const long long total = (long long)A.B * A.Hk * A.rows;
  const Share mine(A.splits);
  const bool on = mine.vector < total * per;
  const long long i = on ? mine.vector : 0, at = fast_div(i, per);
  const int d = (int)(i - at * per) * 8;
  const f32x8 x = mine.sum(A.part + at * A.D + d, total * A.D, A.splits, [](int) { return 1.f; });
  if (!on || mine.first) return;
  const long long bh = at / A.rows;
  const Row row(A, (int)(bh % A.Hk), (int)(at % A.rows));
  *reinterpret_cast<typename Type<T>::x8*>(static_cast<T*>(A.out) + row.packed(A, (int)(bh / A.Hk)) + d) =
      __builtin_convertvector(x * A.scale, typename Type<T>::x8);
}

template <typename T>
__global__ void __launch_bounds__(256) cross_dkv_sum_kernel(const Args A) {
  const long long all = (long long)A.B * A.Lk * A.Hk * A.D;
  const Share mine(A.splits);
  const bool on = mine.vector * 8 < 2 * all;
  const long long i = on ? mine.vector * 8 : 0;
  const f32x8 x = mine.sum(A.part + i, 2 * all, A.splits, [](int) { return 1.f; });
  if (!on || mine.first) return;
  T* o = i < all ? static_cast<T*>(A.dk) + i : static_cast<T*>(A.dv) + (i - all);
  *reinterpret_cast<typename Type<T>::x8*>(o) = __builtin_convertvector(x, typename Type<T>::x8);
}

// ---- the mask as bits: one word per 32 keys, so the kernels read 1/8 of a byte mask's traffic, and that by whole words (40 x 100 x 784: 5.9 us) -----
__global__ void __launch_bounds__(256) cross_pack_kernel(const unsigned char* blocked, long long sb, long long sh, long long sn, long long sk,
                                                         int H, int N, int Lk, int W, long long total, unsigned* bits) {
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= total) return;
  const long long line = fast_div(i, W);
  const int w = (int)(i - line * W);
  const long long bh = fast_div(line, N);
  const long long n = line - bh * N, b = fast_div(bh, H), h = bh - b * H;
  const unsigned char* p = blocked + b * sb + h * sh + n * sn + (long long)w * 32 * sk;
  const int count = min(32, Lk - w * 32);
  unsigned m = 0u;
  if (count == 32 && sk == 1 && ((uintptr_t)p & 15) == 0) {
    const u32x4 x = *reinterpret_cast<const u32x4*>(p), y = *reinterpret_cast<const u32x4*>(p + 16);
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const unsigned word = j < 16 ? x[j >> 2] : y[(j - 16) >> 2];
      m |= ((word >> (8 * (j & 3))) & 0xffu ? 1u : 0u) << j;
    }
  } else {
    for (int j = 0; j < 32; ++j) m |= (j >= count || p[j * sk] ? 1u : 0u) << j;
  }
  bits[i] = m;
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

struct Plan {
  int rows;                   // forward and dq: of a workgroup, 32 (the waves share the keys of a tile) or 128 (a wave has its own)
  int tiles, splits;
  int key_tiles, row_splits;  // dk, dv
};

// Splits of the other axis when there are few workgroups: as many as `slots`, one round of what the chip holds, allow (4 x 10 x 4096 rows against 77
// keys: dk, dv in 13 shares are 520 workgroups and take 26.2 us, in 12 21.8; 3 x 8 x 300 rows over 5000 keys of 128: 24 shares 49.0, 21 38.9).
// Left whole are a walk of a few tiles, which costs no more than the join and saves a launch (8 x 100 rows over 256 keys of 64: 6.1 against 9.7 us
// replayed, 13.6 against 17.3 called; one row of 4 x 8 over 784 keys of 32: 9.1 against 9.6, 13.9 against 18.2; replayed, 8 tiles of 64: 10.8
// against 10.3, 8 of 128: 16.6 against 11.3), and from one workgroup a CU on a short axis: 320 workgroups of 13 tiles take 26.8 us, and in two
// halves 22.7 us and a join of 4.2 us and one more launch.
int pick_splits(long long groups, int tiles, int D, int slots) {
  if (tiles <= (D > 64 ? 4 : 7) || (groups >= 256 && tiles < 32)) return 1;
  long long s = slots / groups;
  if (s > tiles) s = tiles;
  if (s > 128) s = 128;
  return s < 1 ? 1 : (int)s;
}

// Blocks of 128 rows read a key once for all of them; blocks of 32 are four times as many.  So these are taken for 32 rows, and where 128 would
// leave CUs idle or need a join and 32 need none (forward, dq, each with its join, 128 against 32 rows a block): 8 x 8 x 100 rows over 784 keys of 32
// 14.2, 15.0 against 10.7, 12.0 us; 1 x 8 x 1024 over 1500 of 64 23.9, 22.3 against 18.2, 20.6; 2 x 8 x 512 over 1024 of 128 27.5, 30.5 against 20.9,
// 27.8; even at 1 x 8 x 1000 over 2000 of 32 (16.8, 19.0 against 18.0, 19.0, and a launch less) and 1 x 8 x 1024 over 2048 of 128 (35.1, 36.2
// against 35.7, 41.8), and longer walks stay with 128.  Not for dq of more than 64 dimensions, with one workgroup a CU, beyond one round of them:
// 16 x 8 x 100 over 784 of 128 32.0 against 40.4.
Plan plan_of(const combo_cross_attention_t& d, bool back) {
  Plan p;
  const int G = d.Hq / d.Hk;
  const long long rows = (long long)d.Lq * G, bh = (long long)d.B * d.Hk, small = bh * ((rows + 31) / 32);
  const bool whole = bh * ((rows + 127) / 128) < 256 && d.Lk <= (d.D > 64 ? 1024 : 2048) && pick_splits(small, (d.Lk + 127) / 128, d.D, 512) == 1 &&
                     !(back && d.D > 64 && small > 256);
  p.rows = rows <= 32 || whole ? 32 : 128;
  p.tiles = (int)((rows + p.rows - 1) / p.rows);
  const int kt = p.rows == 32 ? 128 : 64, key_tiles = (d.Lk + kt - 1) / kt;
  p.splits = pick_splits(bh * p.tiles, key_tiles, d.D, 512);  // (two workgroups a CU)
  // few rows, which cost what it takes to read the keys: shares of 32 tiles and more are halved, so that the workgroups of the longer samples do
  // not finish alone (16 x 8 x 16384 keys of 128: all as long 208 -> 198 us, 5.4 TB/s; 25 to 100 % as long 165 -> 153; shares of 8 tiles, 8 x 8
  // x 4096 keys: 26.6 against 27.5)
  if (p.rows == 32 && key_tiles >= 32 * p.splits) p.splits *= 2;
  p.key_tiles = (d.Lk + 127) / 128;
  const int slots = d.D > 64 ? 256 : (d.D > 32 ? 512 : 768);  // (one, two, three a CU; 2 x 8 x 512 rows, 1024 keys of 128: 31.4 us in 512, 24.6 in 256)
  p.row_splits = pick_splits(bh * p.key_tiles, (int)((rows + 31) / 32), d.D, slots);
  return p;
}

long long blocks_of(long long items) { return (items + 255) / 256; }

constexpr long long kMaxGrid = 1 << 24;  // workgroups of 256 threads

bool desc_ok(const combo_cross_attention_t* d) {
  if (!d || !d->q || !d->k || !d->v || d->B <= 0 || d->Lq <= 0 || d->Lk <= 0 || d->Hq <= 0 || d->Hk <= 0 || d->Hq % d->Hk || d->D <= 0 || d->D > 128 ||
      d->D % 8 || (d->dtype != 1 && d->dtype != 2) || !(d->scale > 0.f) || !std::isfinite(d->scale * 1.4427f))
    return false;
  if (((uintptr_t)d->q | (uintptr_t)d->k | (uintptr_t)d->v) & 15 || ((uintptr_t)d->kv_lengths | (uintptr_t)d->blocked_bits) & 3) return false;
  for (int i = 0; i < 3; ++i)
    if ((d->q_stride[i] | d->k_stride[i] | d->v_stride[i]) & 7 || d->q_stride[i] < 0 || d->k_stride[i] < 0 || d->v_stride[i] < 0 ||
        d->bits_stride[i] < 0)
      return false;
  if (d->k_stride[1] > (1 << 22) || d->v_stride[1] > (1 << 22)) return false;  // (32-bit byte offsets inside a tile of 128 keys)
  if ((long long)d->Lq * (d->Hq / d->Hk) >= (1ll << 30) || d->Lk >= (1 << 30)) return false;
  for (const bool back : {false, true}) {  // (workgroups of the largest launches: a grid holds less than 2^32 threads)
    const Plan p = plan_of(*d, back);
    if ((long long)d->B * d->Hk * p.tiles * p.splits >= kMaxGrid || (long long)d->B * d->Hk * p.key_tiles * p.row_splits >= kMaxGrid) return false;
  }
  return true;
}

Args args_of(const combo_cross_attention_t& d) {
  Args A = {};
  A.q = static_cast<const char*>(d.q), A.k = static_cast<const char*>(d.k), A.v = static_cast<const char*>(d.v);
  A.qb = d.q_stride[0], A.qn = d.q_stride[1], A.qh = d.q_stride[2];
  A.kb = d.k_stride[0], A.kn = d.k_stride[1], A.kh = d.k_stride[2];
  A.vb = d.v_stride[0], A.vn = d.v_stride[1], A.vh = d.v_stride[2];
  A.lens = d.kv_lengths, A.bits = d.blocked_bits;
  A.mb = d.bits_stride[0], A.mh = d.bits_stride[1], A.mn = d.bits_stride[2];
  A.B = d.B, A.Lq = d.Lq, A.Lk = d.Lk, A.Hq = d.Hq, A.Hk = d.Hk, A.G = d.Hq / d.Hk, A.D = d.D, A.rows = d.Lq * A.G;
  A.scale = d.scale, A.c = d.scale * 1.44269504088896341f;
  return A;
}

template <void (*kernel)(const Args)>
int launch(long long grid, size_t lds, const Args& A, hipStream_t st) {
  if (grid <= 0 || grid >= kMaxGrid) return COMBO_EINVAL;
  if (lds > 65536) {
    static ComboDevFlag ready;  // (one per kernel: it is the template's argument)
    if (!ready.is_set()) {
      const hipError_t rc = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (rc != hipSuccess) return (int)rc;
      ready.mark();
    }
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), lds, st, A);
  return (int)hipGetLastError();
}

template <typename T, int DP>
int forward(Args& A, const Plan& p, hipStream_t st) {
  A.tiles = p.tiles, A.splits = p.splits;
  const long long grid = (long long)A.B * A.Hk * A.splits * A.tiles;
  int rc = p.rows == 32 ? launch<cross_few_kernel<T, DP>>(grid, Few<DP>::LDS, A, st) : launch<cross_wide_kernel<T, DP>>(grid, Wide<DP>::LDS, A, st);
  if (rc == 0 && A.splits > 1) rc = launch<cross_join_kernel<T>>(blocks_of((long long)A.B * A.Hk * A.rows * (A.D / 8) * lanes_of(A.splits)), 0, A, st);
  return rc;
}

template <typename T, int DP>
int backward(Args& A, const Plan& p, hipStream_t st) {
  float* part = A.part;
  A.tiles = p.tiles, A.splits = p.splits;
  const long long grid = (long long)A.B * A.Hk * A.splits * A.tiles;
  int rc = p.rows == 32 ? launch<cross_dq_kernel<T, DP, 1>>(grid, Dq<DP, 1>::LDS, A, st)
                        : launch<cross_dq_kernel<T, DP, 4>>(grid, Dq<DP, 4>::LDS, A, st);
  if (rc == 0 && A.splits > 1)
    rc = launch<cross_dq_sum_kernel<T>>(blocks_of((long long)A.B * A.Hk * A.rows * (A.D / 8) * lanes_of(A.splits)), 0, A, st);
  if (rc) return rc;
  if (!A.dk) return 0;
  A.part = part;
  A.tiles = p.key_tiles, A.splits = p.row_splits;
  rc = launch<cross_dkv_kernel<T, DP>>((long long)A.B * A.Hk * A.splits * A.tiles, Bwd<T, DP>::LDS, A, st);
  if (rc == 0 && A.splits > 1)
    rc = launch<cross_dkv_sum_kernel<T>>(blocks_of((long long)A.B * A.Lk * A.Hk * (A.D / 8) * 2 * lanes_of(A.splits)), 0, A, st);
  return rc;
}

template <typename T>
int by_dim(Args& A, const Plan& p, bool back, hipStream_t st) {
  if (A.D <= 32) return back ? backward<T, 32>(A, p, st) : forward<T, 32>(A, p, st);
  if (A.D <= 64) return back ? backward<T, 64>(A, p, st) : forward<T, 64>(A, p, st);
  return back ? backward<T, 128>(A, p, st) : forward<T, 128>(A, p, st);
}

}  // namespace

extern "C" {

long long combo_cross_attention_workspace(const combo_cross_attention_t* d, int backward_pass) {
  if (!desc_ok(d)) return -1;
  const Plan p = plan_of(*d, backward_pass);
  const long long rows = (long long)d->B * d->Hq * d->Lq;
  if (!backward_pass) return p.splits > 1 ? p.splits * rows * (d->D + 1) * 4 : 0;
  const long long dq = p.splits > 1 ? p.splits * rows * d->D : 0;
  const long long dkv = p.row_splits > 1 ? 2ll * p.row_splits * d->B * d->Lk * d->Hk * d->D : 0;
  return ((dq > dkv ? dq : dkv) + rows) * 4;
}

int combo_cross_attention_forward(const combo_cross_attention_t* d, void* out, float* lse, void* workspace, combo_stream_t stream) {
  if (!desc_ok(d) || !out || ((uintptr_t)out & 15) || ((uintptr_t)lse & 3) || ((uintptr_t)workspace & 31)) return COMBO_EINVAL;
  const Plan p = plan_of(*d, false);
  if (p.splits > 1 && !workspace) return COMBO_EINVAL;
  Args A = args_of(*d);
  A.out = out, A.lse = lse, A.part = static_cast<float*>(workspace);
  if (p.splits > 1) A.part_lse = A.part + (long long)p.splits * d->B * d->Hq * d->Lq * d->D;
  return d->dtype == 1 ? by_dim<__bf16>(A, p, false, (hipStream_t)stream) : by_dim<_Float16>(A, p, false, (hipStream_t)stream);
}

int combo_cross_attention_backward(const combo_cross_attention_t* d, const void* out, const float* lse, const void* dout, void* workspace,
                                   void* dq, void* dk, void* dv, combo_stream_t stream) {
  if (!desc_ok(d) || !out || !lse || !dout || !workspace || !dq || (!dk) != (!dv) ||
      (((uintptr_t)out | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) || ((uintptr_t)lse & 3) || ((uintptr_t)workspace & 31))
    return COMBO_EINVAL;
  const Plan p = plan_of(*d, true);
  Args A = args_of(*d);
  A.o = out, A.lse = const_cast<float*>(lse), A.dout = dout, A.out = dq, A.dk = dk, A.dv = dv;
  const long long bytes = combo_cross_attention_workspace(d, 1);
  A.part = static_cast<float*>(workspace);
  A.delta = A.part + bytes / 4 - (long long)d->B * d->Hq * d->Lq;
  return d->dtype == 1 ? by_dim<__bf16>(A, p, true, (hipStream_t)stream) : by_dim<_Float16>(A, p, true, (hipStream_t)stream);
}

int combo_cross_attention_pack(const unsigned char* blocked, long long stride_b, long long stride_h, long long stride_n, long long stride_k, int B,
                               int H, int N, int Lk, unsigned* bits, combo_stream_t stream) {
  if (!blocked || !bits || B <= 0 || H <= 0 || N <= 0 || Lk <= 0 || stride_b < 0 || stride_h < 0 || stride_n < 0 || stride_k < 0) return COMBO_EINVAL;
  const int W = (Lk + 31) / 32;
  const long long total = (long long)B * H * N * W, grid = blocks_of(total);
  if (grid >= kMaxGrid) return COMBO_EINVAL;
  hipLaunchKernelGGL(cross_pack_kernel, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, blocked, stride_b, stride_h, stride_n, stride_k, H, N,
                     Lk, W, total, bits);
  return (int)hipGetLastError();
}

}  // extern "C"
