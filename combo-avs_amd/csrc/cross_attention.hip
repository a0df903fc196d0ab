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
// and dO are each staged once, row-major, for both uses.  LDS tiles are swizzled in 16-byte chunks (Tile::chunk).
#include <cmath>

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

// row-major LDS tile of 16-bit values, DP a row, in chunks of 8: chunk c of row r lies at chunk c ^ swizzle(r).  16 rows at the same chunk
// (a b128 operand read) and 4 rows x 4 neighbouring chunks (a transposed read) then both spread over all banks: the swizzle is the bit
// reversal of the row's index among those that start at the same bank.
template <int DP>
struct Tile {
  static constexpr int CH = DP / 8, PER = 16 / CH;  // chunks of a row; rows over which the banks repeat
  static __device__ __forceinline__ int swizzle(int r) {
    const int x = (r / PER) & (CH - 1);
    if constexpr (CH == 4) return x;
    if constexpr (CH == 8) return ((x & 1) << 2) | (x & 2) | ((x >> 2) & 1);
    return ((x & 1) << 3) | ((x & 2) << 1) | ((x & 4) >> 1) | ((x >> 3) & 1);
  }
  static __device__ __forceinline__ int at(int r, int c) { return r * DP + ((c ^ swizzle(r)) << 3); }
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
  const T* a = tile + Tile<DP>::at(row, col >> 3) + (col & 7);
  const T* b = tile + Tile<DP>::at(row + 8, col >> 3) + (col & 7);
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

__device__ __forceinline__ float other_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// index of register i of a 32 x 32 result along its rows
__device__ __forceinline__ int reg_row(int i, int half) { return 8 * (i >> 2) + 4 * half + (i & 3); }

// ROWS rows of DP values from global memory into registers and on into an LDS tile; rows from `valid` on, chunks from D on and rows whose bit
// is set in `skip` (blocked for every query: whatever such a state holds never meets a product) become zeros
template <typename T, int DP, int ROWS>
struct Stage {
  static constexpr int N = ROWS * (DP / 8) / 256;
  u32x4 r[N];
  __device__ __forceinline__ void load(const T* base, long long stride, int row0, int valid, int D, const unsigned* skip) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = threadIdx.x + 256 * i, row = row0 + x / (DP / 8), c = x % (DP / 8);
      bool on = row < valid && c * 8 < D;
      if (skip && on) on = !((skip[row >> 5] >> (row & 31)) & 1);
      u32x4 z = {0u, 0u, 0u, 0u};
      if (on) z = *reinterpret_cast<const u32x4*>(base + row * stride + c * 8);
      r[i] = z;
    }
  }
  __device__ __forceinline__ void store(T* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = threadIdx.x + 256 * i, row = x / (DP / 8), c = x % (DP / 8);
      *reinterpret_cast<u32x4*>(tile + Tile<DP>::at(row, c)) = r[i];
    }
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

// scores of keys key0 .. key0 + 31 against this lane's row: lengths and mask
__device__ __forceinline__ void mask_scores(f32x16& s, int key0, int len, const unsigned* words, int half) {
  if (key0 + 32 > len) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (key0 + reg_row(i, half) >= len) s[i] = -kInf;
  }
  if (words) {
    const unsigned w = (key0 < len ? words[key0 >> 5] : 0xffffffffu) >> (4 * half);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (w & (1u << (8 * (i >> 2) + (i & 3)))) s[i] = -kInf;
  }
}

struct Range { int lo, hi; };
// the keys of split `s`: whole tiles of the sample's own length
__device__ __forceinline__ Range split_range(int len, int splits, int s, int tile) {
  const int tiles = (len + tile - 1) / tile, per = (tiles + splits - 1) / splits;
  return {min(len, s * per * tile), min(len, (s + 1) * per * tile)};
}

// ---- forward ------------------------------------------------------------------------------------------------------------------

// RW waves along the rows (32 each), 4 / RW along the keys of a tile
template <typename T, int DP, int RW>
struct Fwd {
  static constexpr int KW = 4 / RW, KB = RW == 4 ? 2 : 1, KT = 32 * KB * KW, RT = 32 * RW;
  static constexpr int LDS = 2 * KT * DP * 2 + (KW > 1 ? 2 * KW * 32 * 4 : 0);
  static_assert(KW == 1 || KW * 32 * DP * 4 <= 2 * KT * DP * 2, "the join of the key waves fits the tiles");
};

template <typename T, int DP, int RW>
__global__ void __launch_bounds__(256) cross_forward_kernel(const Args A) {
  typedef Fwd<T, DP, RW> F;
  typedef typename Type<T>::x8 x8;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* Kt = reinterpret_cast<T*>(lds);
  T* Vt = Kt + F::KT * DP;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int rw = wave % RW, kw = wave / RW;
  int id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int tile = id % A.tiles;
  id /= A.tiles;
  const int split = id % A.splits;
  id /= A.splits;
  const int hk = id % A.Hk, b = id / A.Hk;
  const int r = tile * F::RT + rw * 32 + (lane & 31), len = length_of(A, b);
  const Row row(A, hk, min(r, A.rows - 1));
  const Range keys = split_range(len, A.splits, split, F::KT);
  const T* k = reinterpret_cast<const T*>(A.k) + b * A.kb + hk * A.kh;
  const T* v = reinterpret_cast<const T*>(A.v) + b * A.vb + hk * A.vh;
  const unsigned* words = A.bits ? A.bits + b * A.mb + row.h * A.mh + row.n * A.mn : nullptr;
  const unsigned* skip = A.bits && A.mn == 0 && (A.mh == 0 || A.G == 1) ? A.bits + b * A.mb + hk * A.mh : nullptr;
  x8 q[DP / 16];
  row_operand<T, DP>(reinterpret_cast<const T*>(A.q) + b * A.qb + row.n * A.qn + row.h * A.qh, A.D, r < A.rows, q);
  f32x16 acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
  float m = -kInf, l = 0.f;
  Stage<T, DP, F::KT> sk, sv;
  for (int k0 = keys.lo; k0 < keys.hi; k0 += F::KT) {
    sk.load(k, A.kn, k0, len, A.D, skip);
    sv.load(v, A.vn, k0, len, A.D, skip);
    __syncthreads();
    sk.store(Kt);
    sv.store(Vt);
    __syncthreads();
    f32x16 s[F::KB];
#pragma unroll
    for (int kb = 0; kb < F::KB; ++kb) {
      const int row0 = (kw * F::KB + kb) * 32;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) s[kb] = Type<T>::mfma(operand<T, DP>(Kt, row0, d), q[d], s[kb]);
      mask_scores(s[kb], k0 + row0, len, words, half);
    }
    float top = m;
#pragma unroll
    for (int kb = 0; kb < F::KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kb][i]);
    top = other_max(top);
    const float base = top == -kInf ? 0.f : top * A.c;
    const float alpha = __builtin_amdgcn_exp2f(m * A.c - base);  // (m = -inf: 0)
    m = top;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] *= alpha;
#pragma unroll
    for (int kb = 0; kb < F::KB; ++kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[kb][i] = __builtin_amdgcn_exp2f(fmaf(s[kb][i], A.c, -base));
        l += s[kb][i];
      }
      // p is rounded to the tensor's type for the product (half a step relative to each p); its sum l keeps 32 bits
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const x8 p = pack<T>(s[kb], st);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] = Type<T>::mfma(operand_t<T, DP>(Vt, (kw * F::KB + kb) * 32 + 16 * st, 32 * d), p, acc[d]);
      }
    }
  }
  l = both_sum(l);
  float lse;
  if constexpr (F::KW > 1) {  // the key waves hold the same rows: join their maxima, sums and results
    float* ml = reinterpret_cast<float*>(lds + 2 * F::KT * DP * 2);
    float* part = reinterpret_cast<float*>(lds);  // [KW][DP][32]
    __syncthreads();
    if (half == 0) {
      ml[kw * 32 + lane] = m;
      ml[(F::KW + kw) * 32 + lane] = l;
    }
    __syncthreads();
    float top = -kInf, sum = 0.f;
#pragma unroll
    for (int w = 0; w < F::KW; ++w) top = fmaxf(top, ml[w * 32 + (lane & 31)]);
    const float base = top == -kInf ? 0.f : top * A.c;
#pragma unroll
    for (int w = 0; w < F::KW; ++w)
      sum += ml[(F::KW + w) * 32 + (lane & 31)] * __builtin_amdgcn_exp2f(ml[w * 32 + (lane & 31)] * A.c - base);
    const float f = sum > 0.f ? __builtin_amdgcn_exp2f(m * A.c - base) / sum : (sum == 0.f ? 0.f : sum);
    lse = sum > 0.f ? base + log2f(sum) : (sum == 0.f ? -kInf : sum);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) part[(kw * DP + 32 * d + reg_row(i, half)) * 32 + (lane & 31)] = acc[d][i] * f;
    __syncthreads();
    // wave w gathers its share of the dimensions
    if (r < A.rows) {
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
        if (d < A.D) {
          if (A.splits > 1) {
            float* o = A.part + ((((long long)split * A.B + b) * A.Hk + hk) * A.rows + r) * A.D + d;
            *reinterpret_cast<float4*>(o) = make_float4(x[0], x[1], x[2], x[3]);
          } else {
            typename Type<T>::x4 y;
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = (T)x[j];
            *reinterpret_cast<typename Type<T>::x4*>(static_cast<T*>(A.out) + row.packed(A, b) + d) = y;
          }
        }
      }
    }
    if (kw != 0) return;
  } else {
    const float base = m == -kInf ? 0.f : m * A.c;
    const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    lse = l > 0.f ? base + log2f(l) : (l == 0.f ? -kInf : l);
    if (r < A.rows) {
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int dd = 32 * d + reg_row(i, half);
          if (dd < A.D) {
            if (A.splits > 1) {
              float* o = A.part + ((((long long)split * A.B + b) * A.Hk + hk) * A.rows + r) * A.D + dd;
              *reinterpret_cast<float4*>(o) = make_float4(acc[d][i] * f, acc[d][i + 1] * f, acc[d][i + 2] * f, acc[d][i + 3] * f);
            } else {
              typename Type<T>::x4 y;
#pragma unroll
              for (int j = 0; j < 4; ++j) y[j] = (T)(acc[d][i + j] * f);
              *reinterpret_cast<typename Type<T>::x4*>(static_cast<T*>(A.out) + row.packed(A, b) + dd) = y;
            }
          }
        }
    }
  }
  if (half == 0 && r < A.rows) {
    const long long at = ((long long)b * A.Hk + hk) * A.rows + r;
    if (A.splits > 1) A.part_lse[split * ((long long)A.B * A.Hk * A.rows) + at] = lse;
    else if (A.lse) A.lse[at] = lse == -kInf ? kInf : lse;  // (+inf: the backward pass finds p = 0)
  }
}

// joins the splits of a row: 8 values a thread
template <typename T>
__global__ void __launch_bounds__(256) cross_join_kernel(const Args A) {
  const int per = A.D / 8;
  const long long total = (long long)A.B * A.Hk * A.rows, i = blockIdx.x * 256ll + threadIdx.x;
  const long long at = fast_div(i, per);
  if (at >= total) return;
  const int d = (int)(i - at * per) * 8;
  float top = -kInf, sum = 0.f;
  for (int s = 0; s < A.splits; ++s) top = fmaxf(top, A.part_lse[s * total + at]);
  const float base = top == -kInf ? 0.f : top;
  f32x8 x = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < A.splits; ++s) {
    const float w = __builtin_amdgcn_exp2f(A.part_lse[s * total + at] - base);
    sum += w;
    const f32x8 y = *reinterpret_cast<const f32x8*>(A.part + (s * total + at) * A.D + d);
    x += y * w;
  }
  const float f = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  const int r = (int)(at % A.rows);
  const long long bh = at / A.rows;
  const int hk = (int)(bh % A.Hk), b = (int)(bh / A.Hk);
  const Row row(A, hk, r);
  *reinterpret_cast<typename Type<T>::x8*>(static_cast<T*>(A.out) + row.packed(A, b) + d) = __builtin_convertvector(x * f, typename Type<T>::x8);
  if (A.lse && d == 0) A.lse[at] = sum > 0.f ? base + log2f(sum) : (sum == 0.f ? kInf : sum);
}

// ---- backward -----------------------------------------------------------------------------------------------------------------

// dq: the forward's walk over the keys; two score-sized products and the one with K
template <typename T, int DP, int RW>
__global__ void __launch_bounds__(256) cross_dq_kernel(const Args A) {
  typedef Fwd<T, DP, RW> F;
  typedef typename Type<T>::x8 x8;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* Kt = reinterpret_cast<T*>(lds);
  T* Vt = Kt + F::KT * DP;
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
  const Row row(A, hk, min(r, A.rows - 1));
  const Range keys = split_range(len, A.splits, split, F::KT);
  const T* k = reinterpret_cast<const T*>(A.k) + b * A.kb + hk * A.kh;
  const T* v = reinterpret_cast<const T*>(A.v) + b * A.vb + hk * A.vh;
  const unsigned* words = A.bits ? A.bits + b * A.mb + row.h * A.mh + row.n * A.mn : nullptr;
  const unsigned* skip = A.bits && A.mn == 0 && (A.mh == 0 || A.G == 1) ? A.bits + b * A.mb + hk * A.mh : nullptr;
  const long long at = ((long long)b * A.Hk + hk) * A.rows + r;
  x8 q[DP / 16], g[DP / 16];
  row_operand<T, DP>(reinterpret_cast<const T*>(A.q) + b * A.qb + row.n * A.qn + row.h * A.qh, A.D, on, q);
  row_operand<T, DP>(static_cast<const T*>(A.dout) + row.packed(A, b), A.D, on, g);
  float delta = 0.f;
  {  // do . o as the diagonal of a product: the same order of summation as do . v, so a row that sees one key has ds = 0 exactly
    x8 o[DP / 16];
    row_operand<T, DP>(static_cast<const T*>(A.o) + row.packed(A, b), A.D, on, o);
    f32x16 x;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 0.f;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) x = Type<T>::mfma(o[d], g[d], x);
    const int c = lane & 31;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (4 * (c >> 3) + (c & 3) == i) delta = x[i];
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(delta), __float_as_uint(delta), false, false);
    delta = __uint_as_float((c >> 2) & 1 ? sw[1] : sw[0]);
  }
  const float lse = on ? A.lse[at] : kInf;
  if (on && half == 0 && kw == 0 && split == 0) A.delta[at] = delta;
  f32x16 acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
  Stage<T, DP, F::KT> sk, sv;
  for (int k0 = keys.lo; k0 < keys.hi; k0 += F::KT) {
    sk.load(k, A.kn, k0, len, A.D, skip);
    sv.load(v, A.vn, k0, len, A.D, skip);
    __syncthreads();
    sk.store(Kt);
    sv.store(Vt);
    __syncthreads();
#pragma unroll
    for (int kb = 0; kb < F::KB; ++kb) {
      const int row0 = (kw * F::KB + kb) * 32;
      f32x16 s, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = dp[i] = 0.f;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) s = Type<T>::mfma(operand<T, DP>(Kt, row0, d), q[d], s);
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) dp = Type<T>::mfma(operand<T, DP>(Vt, row0, d), g[d], dp);
      mask_scores(s, k0 + row0, len, words, half);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[i], A.c, -lse));
        s[i] = p == 0.f ? 0.f : p * (dp[i] - delta);  // (a blocked key's dp may be anything)
      }
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const x8 ds = pack<T>(s, st);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] = Type<T>::mfma(operand_t<T, DP>(Kt, row0 + 16 * st, 32 * d), ds, acc[d]);
      }
    }
  }
  auto store = [&](int d, const float (&x)[4]) {
    if (d >= A.D) return;
    if (A.splits > 1) {
      float* o = A.part + ((((long long)split * A.B + b) * A.Hk + hk) * A.rows + r) * A.D + d;
      *reinterpret_cast<float4*>(o) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
      typename Type<T>::x4 y;
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = (T)(x[j] * A.scale);
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
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const float x[4] = {acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]};
        store(32 * d + reg_row(i, half), x);
      }
  }
}

// sums the splits of dq
template <typename T>
__global__ void __launch_bounds__(256) cross_dq_sum_kernel(const Args A) {
  const int per = A.D / 8;
  const long long total = (long long)A.B * A.Hk * A.rows, i = blockIdx.x * 256ll + threadIdx.x;
  const long long at = fast_div(i, per);
  if (at >= total) return;
  const int d = (int)(i - at * per) * 8;
  f32x8 x = *reinterpret_cast<const f32x8*>(A.part + at * A.D + d);
  for (int s = 1; s < A.splits; ++s) x += *reinterpret_cast<const f32x8*>(A.part + (s * total + at) * A.D + d);
  const int r = (int)(at % A.rows);
  const long long bh = at / A.rows;
  const Row row(A, (int)(bh % A.Hk), r);
  *reinterpret_cast<typename Type<T>::x8*>(static_cast<T*>(A.out) + row.packed(A, (int)(bh / A.Hk)) + d) =
      __builtin_convertvector(x * A.scale, typename Type<T>::x8);
}

// dk, dv: a wave owns 32 keys, the workgroup walks the rows of all G heads.  Score tiles are rows x keys here (a lane owns a key), so they are
// the B operands of dV^T = dO^T P and dK^T = Q^T dS; lse and delta of a tile's rows lie in LDS.
template <typename T, int DP>
struct Bwd {
  static constexpr int KT = 128, RT = 64 * 64 / DP < 32 ? 32 : (64 * 64 / DP > 64 ? 64 : 64 * 64 / DP);
  static constexpr int LDS = 2 * RT * DP * 2 + 2 * RT * 4 + 4 * RT * 4;
};

template <typename T, int DP>
__global__ void __launch_bounds__(256) cross_dkv_kernel(const Args A) {
  typedef Bwd<T, DP> F;
  typedef typename Type<T>::x8 x8;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* Qt = reinterpret_cast<T*>(lds);
  T* Gt = Qt + F::RT * DP;
  float* Lt = reinterpret_cast<float*>(Gt + F::RT * DP);
  float* Dt = Lt + F::RT;
  unsigned* Mt = reinterpret_cast<unsigned*>(Dt + F::RT);  // [4 waves][RT]: the mask words of the wave's keys
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
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) ak[d][i] = av[d][i] = 0.f;
  const int row_tiles = (A.rows + F::RT - 1) / F::RT, per = (row_tiles + A.splits - 1) / A.splits;
  const int lo = split * per, hi = tile * F::KT < len ? min(row_tiles, (split + 1) * per) : lo;
  const T* q = reinterpret_cast<const T*>(A.q) + b * A.qb;
  const T* g = static_cast<const T*>(A.dout);
  for (int rt = lo; rt < hi; ++rt) {
    constexpr int N = F::RT * (DP / 8) / 256;
    u32x4 rq[N], rg[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = threadIdx.x + 256 * i, r = rt * F::RT + x / (DP / 8), c = x % (DP / 8);
      u32x4 z = {0u, 0u, 0u, 0u};
      rq[i] = rg[i] = z;
      if (r < A.rows && c * 8 < A.D) {
        const Row row(A, hk, r);
        rq[i] = *reinterpret_cast<const u32x4*>(q + row.n * A.qn + row.h * A.qh + c * 8);
        rg[i] = *reinterpret_cast<const u32x4*>(g + row.packed(A, b) + c * 8);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = threadIdx.x + 256 * i, at = Tile<DP>::at(x / (DP / 8), x % (DP / 8));
      *reinterpret_cast<u32x4*>(Qt + at) = rq[i];
      *reinterpret_cast<u32x4*>(Gt + at) = rg[i];
    }
    if (threadIdx.x < F::RT) {
      const int r = rt * F::RT + threadIdx.x;
      const long long at = ((long long)b * A.Hk + hk) * A.rows + r;
      Lt[threadIdx.x] = r < A.rows ? A.lse[at] : kInf;
      Dt[threadIdx.x] = r < A.rows ? A.delta[at] : 0.f;
    }
    if (A.bits) {
      for (int x = threadIdx.x; x < 4 * F::RT; x += 256) {
        const int r = rt * F::RT + x % F::RT, w = tile * 4 + x / F::RT;
        unsigned m = 0xffffffffu;
        if (r < A.rows && w * 32 < A.Lk) {
          const Row row(A, hk, r);
          m = A.bits[b * A.mb + row.h * A.mh + row.n * A.mn + w];
        }
        Mt[x] = m;
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int rb = 0; rb < F::RT; rb += 32) {
      f32x16 s, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = dp[i] = 0.f;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) s = Type<T>::mfma(operand<T, DP>(Qt, rb, d), k[d], s);
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) dp = Type<T>::mfma(operand<T, DP>(Gt, rb, d), v[d], dp);
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const float4 L = *reinterpret_cast<const float4*>(Lt + rb + reg_row(i, half));
        s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], A.c, -L.x));
        s[i + 1] = __builtin_amdgcn_exp2f(fmaf(s[i + 1], A.c, -L.y));
        s[i + 2] = __builtin_amdgcn_exp2f(fmaf(s[i + 2], A.c, -L.z));
        s[i + 3] = __builtin_amdgcn_exp2f(fmaf(s[i + 3], A.c, -L.w));
      }
      if (A.bits) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const uint4 w = *reinterpret_cast<const uint4*>(Mt + wave * F::RT + rb + reg_row(i, half));
          const unsigned bit = 1u << (lane & 31);
          if (w.x & bit) s[i] = 0.f;
          if (w.y & bit) s[i + 1] = 0.f;
          if (w.z & bit) s[i + 2] = 0.f;
          if (w.w & bit) s[i + 3] = 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const float4 X = *reinterpret_cast<const float4*>(Dt + rb + reg_row(i, half));
        dp[i] = s[i] == 0.f ? 0.f : s[i] * (dp[i] - X.x);
        dp[i + 1] = s[i + 1] == 0.f ? 0.f : s[i + 1] * (dp[i + 1] - X.y);
        dp[i + 2] = s[i + 2] == 0.f ? 0.f : s[i + 2] * (dp[i + 2] - X.z);
        dp[i + 3] = s[i + 3] == 0.f ? 0.f : s[i + 3] * (dp[i + 3] - X.w);
      }
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const x8 p = pack<T>(s, st), ds = pack<T>(dp, st);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          av[d] = Type<T>::mfma(operand_t<T, DP>(Gt, rb + 16 * st, 32 * d), p, av[d]);
          ak[d] = Type<T>::mfma(operand_t<T, DP>(Qt, rb + 16 * st, 32 * d), ds, ak[d]);
        }
      }
    }
  }
  if (key >= A.Lk) return;
  const bool mine = open;  // (keys behind the length or blocked for all: zeros)
  const long long at = (((long long)b * A.Lk + key) * A.Hk + hk) * A.D, all = (long long)A.B * A.Lk * A.Hk * A.D;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int dd = 32 * d + reg_row(i, half);
      if (dd >= A.D) continue;
      float x[4], y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = mine ? ak[d][i + j] * A.scale : 0.f;
        y[j] = mine ? av[d][i + j] : 0.f;
      }
      if (A.splits > 1) {
        float* o = A.part + 2 * split * all + at + dd;
        *reinterpret_cast<float4*>(o) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(o + all) = make_float4(y[0], y[1], y[2], y[3]);
      } else {
        typename Type<T>::x4 a, c;
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = (T)x[j], c[j] = (T)y[j];
        *reinterpret_cast<typename Type<T>::x4*>(static_cast<T*>(A.dk) + at + dd) = a;
        *reinterpret_cast<typename Type<T>::x4*>(static_cast<T*>(A.dv) + at + dd) = c;
      }
    }
}

// sums the splits of dk and dv: 8 values a thread
template <typename T>
__global__ void __launch_bounds__(256) cross_dkv_sum_kernel(const Args A) {
  const long long all = (long long)A.B * A.Lk * A.Hk * A.D, i = (blockIdx.x * 256ll + threadIdx.x) * 8;
  if (i >= 2 * all) return;
  f32x8 x = *reinterpret_cast<const f32x8*>(A.part + i);
  for (int s = 1; s < A.splits; ++s) x += *reinterpret_cast<const f32x8*>(A.part + 2 * s * all + i);
  T* o = i < all ? static_cast<T*>(A.dk) + i : static_cast<T*>(A.dv) + (i - all);
  *reinterpret_cast<typename Type<T>::x8*>(o) = __builtin_convertvector(x, typename Type<T>::x8);
}

// ---- the mask as bits: one word per 32 keys, so the kernels read 1/8 of a byte mask's traffic, and that by whole words ----------
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
  int narrow, tiles, splits;        // forward and dq
  int key_tiles, row_splits;        // dk, dv
};

int pick_splits(long long groups, int tiles) {
  // two workgroups for each of the 256 CUs; a split has at least one tile
  long long s = (512 + groups - 1) / groups;
  if (s > tiles) s = tiles;
  if (s > 128) s = 128;
  return s < 1 ? 1 : (int)s;
}

Plan plan_of(const combo_cross_attention_t& d) {
  Plan p;
  const int G = d.Hq / d.Hk;
  const long long rows = (long long)d.Lq * G, bh = (long long)d.B * d.Hk;
  p.narrow = rows <= 32;
  p.tiles = p.narrow ? 1 : (int)((rows + 127) / 128);
  const int kt = p.narrow ? 128 : 64;
  p.splits = pick_splits(bh * p.tiles, (d.Lk + kt - 1) / kt);
  p.key_tiles = (d.Lk + 127) / 128;
  p.row_splits = pick_splits(bh * p.key_tiles, (int)((rows + 31) / 32));
  return p;
}

bool desc_ok(const combo_cross_attention_t* d) {
  if (!d || !d->q || !d->k || !d->v || d->B <= 0 || d->Lq <= 0 || d->Lk <= 0 || d->Hq <= 0 || d->Hk <= 0 || d->Hq % d->Hk || d->D <= 0 || d->D > 128 ||
      d->D % 8 || (d->dtype != 1 && d->dtype != 2) || !(d->scale > 0.f) || !std::isfinite(d->scale))
    return false;
  if (((uintptr_t)d->q | (uintptr_t)d->k | (uintptr_t)d->v) & 15) return false;
  for (int i = 0; i < 3; ++i)
    if ((d->q_stride[i] | d->k_stride[i] | d->v_stride[i]) & 7 || d->q_stride[i] < 0 || d->k_stride[i] < 0 || d->v_stride[i] < 0) return false;
  const long long G = d->Hq / d->Hk;
  return (long long)d->Lq * G < (1ll << 30) && d->Lk < (1 << 30) && (long long)d->B * d->Hq * (((long long)d->Lq + 127) / 128 + ((long long)d->Lk + 127) / 128) < (1 << 24);
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
  if (grid <= 0 || grid > 0x7fffffffll) return COMBO_EINVAL;
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

long long blocks_of(long long items) { return (items + 255) / 256; }

template <typename T, int DP>
int forward(Args& A, const Plan& p, hipStream_t st) {
  A.tiles = p.tiles, A.splits = p.splits;
  const long long grid = (long long)A.B * A.Hk * A.splits * A.tiles;
  int rc = p.narrow ? launch<cross_forward_kernel<T, DP, 1>>(grid, Fwd<T, DP, 1>::LDS, A, st)
                    : launch<cross_forward_kernel<T, DP, 4>>(grid, Fwd<T, DP, 4>::LDS, A, st);
  if (rc == 0 && A.splits > 1) rc = launch<cross_join_kernel<T>>(blocks_of((long long)A.B * A.Hk * A.rows * (A.D / 8)), 0, A, st);
  return rc;
}

template <typename T, int DP>
int backward(Args& A, const Plan& p, hipStream_t st) {
  float* part = A.part;
  A.tiles = p.tiles, A.splits = p.splits;
  const long long grid = (long long)A.B * A.Hk * A.splits * A.tiles;
  int rc = p.narrow ? launch<cross_dq_kernel<T, DP, 1>>(grid, Fwd<T, DP, 1>::LDS, A, st)
                    : launch<cross_dq_kernel<T, DP, 4>>(grid, Fwd<T, DP, 4>::LDS, A, st);
  if (rc == 0 && A.splits > 1) rc = launch<cross_dq_sum_kernel<T>>(blocks_of((long long)A.B * A.Hk * A.rows * (A.D / 8)), 0, A, st);
  if (rc) return rc;
  if (!A.dk) return 0;
  A.part = part;
  A.tiles = p.key_tiles, A.splits = p.row_splits;
  rc = launch<cross_dkv_kernel<T, DP>>((long long)A.B * A.Hk * A.splits * A.tiles, Bwd<T, DP>::LDS, A, st);
  if (rc == 0 && A.splits > 1) rc = launch<cross_dkv_sum_kernel<T>>(blocks_of((long long)A.B * A.Lk * A.Hk * (A.D / 8) * 2), 0, A, st);
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
  const Plan p = plan_of(*d);
  const long long rows = (long long)d->B * d->Hq * d->Lq;
  const long long fwd = p.splits > 1 ? p.splits * rows * (d->D + (backward_pass ? 0 : 1)) : 0;
  if (!backward_pass) return fwd * 4;
  const long long dkv = p.row_splits > 1 ? 2ll * p.row_splits * d->B * d->Lk * d->Hk * d->D : 0;
  return ((fwd > dkv ? fwd : dkv) + rows) * 4;
}

int combo_cross_attention_forward(const combo_cross_attention_t* d, void* out, float* lse, void* workspace, combo_stream_t stream) {
  if (!desc_ok(d) || !out || ((uintptr_t)out & 15) || ((uintptr_t)workspace & 31)) return COMBO_EINVAL;
  const Plan p = plan_of(*d);
  if (p.splits > 1 && !workspace) return COMBO_EINVAL;
  Args A = args_of(*d);
  A.out = out, A.lse = lse, A.part = static_cast<float*>(workspace);
  if (p.splits > 1) A.part_lse = A.part + (long long)p.splits * d->B * d->Hq * d->Lq * d->D;
  return d->dtype == 1 ? by_dim<__bf16>(A, p, false, (hipStream_t)stream) : by_dim<_Float16>(A, p, false, (hipStream_t)stream);
}

int combo_cross_attention_backward(const combo_cross_attention_t* d, const void* out, const float* lse, const void* dout, void* workspace,
                                   void* dq, void* dk, void* dv, combo_stream_t stream) {
  if (!desc_ok(d) || !out || !lse || !dout || !workspace || !dq || (!dk) != (!dv) ||
      (((uintptr_t)out | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) || ((uintptr_t)workspace & 31))
    return COMBO_EINVAL;
  const Plan p = plan_of(*d);
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
  if (grid > 0x7fffffffll) return COMBO_EINVAL;
  hipLaunchKernelGGL(cross_pack_kernel, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, blocked, stride_b, stride_h, stride_n, stride_k, H, N,
                     Lk, W, total, bits);
  return (int)hipGetLastError();
}

}  // extern "C"
