// Rotary positions over several axes (frame, row, column of a video's tokens, or any other): the first 2 P values of a head are P
// pairs, pair j belongs to one axis and is turned by the angle position[axis(j)] * frequency[j]:
//     (lo, hi) -> (lo cos a - hi sin a, hi cos a + lo sin a);    values behind the pairs pass through.
// The gradient is the same kernel with the angle negated.
//
// Bound: HBM (every value is read and written once; 3 flops per value).  The angle of a (token, pair) is shared by all heads, so a
// workgroup first fills an LDS table [tokens][D / 2] of (cos, sin) for its few tokens and then streams all their heads through it:
// the double-precision angle below costs ~60 vector instructions per pair, which per element instead of per (token, pair) would take
// longer than the memory traffic.  Angles in 64 bits: position * frequency is formed in TURNS and reduced to [-1/2, 1/2] in double
// (a position of 1e6 has 3 decimal digits of angle left in fp32); the reduced turn is rounded to fp32 (2^-25 of a turn, 2e-7 rad)
// and goes through sincospi.  The products are fp32, rounded once to the tensor's type.
// 8 x 15680 tokens of 8 x 32 bf16 (64 MB read, 64 written): 28 us = 4.6 TB/s; one token of 8 sequences, or 2 x 713: 4 us, a launch and the angles.
#include "combo_common.h"

namespace {

constexpr int kMaxPairs = 128, kMaxAxes = 8, kTableBytes = 16384;

struct RotaryArgs {
  const char* x;
  char* y;
  const void* pos;
  long long xb, xn, xh;      // strides of x in elements (last dimension contiguous); y is contiguous
  long long pb, pn, pa;      // strides of the positions
  long long tokens;          // B * N
  int N, H, D, P, interleaved, inverse, pos_type;
  int T;                     // tokens per workgroup
  int items;                 // per token: H * per_head
  int per_head;              // vectors of work per head (a lo / hi pair of vectors, or one vector)
  unsigned items_magic, head_magic;
  unsigned char axis[kMaxPairs];
  double turns[kMaxPairs];   // frequency / 2 pi
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec { T v[V]; };

__device__ __forceinline__ double position(const RotaryArgs& A, long long i) {
  switch (A.pos_type) {
    case 0: return (double)static_cast<const float*>(A.pos)[i];
    case 1: return static_cast<const double*>(A.pos)[i];
    case 2: return (double)static_cast<const int*>(A.pos)[i];
    default: return (double)static_cast<const long long*>(A.pos)[i];
  }
}

// n / d for n * d < 2^32 with magic = ceil(2^32 / d) (the launcher keeps items * T below 2^16, heads * vectors below 2^24 with at most
// 256 vectors a head); d = 1 has no 32-bit magic
__device__ __forceinline__ unsigned quick_div(unsigned n, unsigned magic) { return magic ? __umulhi(n, magic) : n; }

template <typename T, int V>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs A) {
  extern __shared__ float2 table[];  // [T][D / 2]; behind the pairs, where an interleaved vector may straddle the border, not used
  const long long t0 = (long long)blockIdx.x * A.T;
  const int nt = (int)min((long long)A.T, A.tokens - t0), half = A.D >> 1;
  for (int i = threadIdx.x; i < nt * half; i += 256) {
    const int t = i / half, j = i - t * half;
    float c = 1.f, s = 0.f;
    if (j < A.P) {
      const long long tok = t0 + t, b = tok / A.N, n = tok - b * A.N;
      double a = position(A, b * A.pb + n * A.pn + A.axis[j] * A.pa) * A.turns[j];
      a -= rint(a);
      sincospif(2.f * (float)a, &s, &c);
      if (A.inverse) s = -s;
    }
    table[i] = make_float2(c, s);
  }
  __syncthreads();
  const T* x = reinterpret_cast<const T*>(A.x);
  T* y = reinterpret_cast<T*>(A.y);
  const int total = nt * A.items, rot = A.P / V;
  for (int i = threadIdx.x; i < total; i += 256) {
    const int t = nt == 1 ? 0 : quick_div(i, A.items_magic), r = i - t * A.items;
    const int h = quick_div(r, A.head_magic), c = r - h * A.per_head;
    const long long tok = t0 + t, b = fast_div(tok, A.N), n = tok - b * A.N;
    const T* src = x + b * A.xb + n * A.xn + h * A.xh;
    T* dst = y + (tok * A.H + h) * A.D;
    const float2* cs = table + t * half;
    if (A.interleaved) {
      const Vec<T, V> a = *reinterpret_cast<const Vec<T, V>*>(src + c * V);
      Vec<T, V> o;
      if constexpr (V >= 2) {
#pragma unroll
        for (int k = 0; k < V; k += 2) {
          const float2 w = cs[(c * V + k) >> 1];
          const float lo = (float)a.v[k], hi = (float)a.v[k + 1];
          const bool turned = c * V + k < 2 * A.P;  // (behind the pairs: as they are, an Inf times the identity's zero would reach its neighbour)
          o.v[k] = turned ? (T)(lo * w.x - hi * w.y) : a.v[k];
          o.v[k + 1] = turned ? (T)(hi * w.x + lo * w.y) : a.v[k + 1];
        }
      }
      *reinterpret_cast<Vec<T, V>*>(dst + c * V) = o;
    } else if (c < rot) {
      const int j = c * V;
      const Vec<T, V> a = *reinterpret_cast<const Vec<T, V>*>(src + j), b2 = *reinterpret_cast<const Vec<T, V>*>(src + A.P + j);
      Vec<T, V> o, o2;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float2 w = cs[j + k];
        const float lo = (float)a.v[k], hi = (float)b2.v[k];
        o.v[k] = (T)(lo * w.x - hi * w.y);
        o2.v[k] = (T)(hi * w.x + lo * w.y);
      }
      *reinterpret_cast<Vec<T, V>*>(dst + j) = o;
      *reinterpret_cast<Vec<T, V>*>(dst + A.P + j) = o2;
    } else {
      const int j = 2 * A.P + (c - rot) * V;
      *reinterpret_cast<Vec<T, V>*>(dst + j) = *reinterpret_cast<const Vec<T, V>*>(src + j);
    }
  }
}

template <typename T>
int launch(RotaryArgs& A, hipStream_t st) {
  // the widest vector (<= 16 bytes) that divides every stride and border the kernel steps by
  const unsigned long long steps = (unsigned long long)A.xb | A.xn | A.xh | (unsigned long long)A.D | ((uintptr_t)A.x | (uintptr_t)A.y) / sizeof(T) |
                                   (A.interleaved ? 0u : (unsigned)A.P);
  int V = 16 / (int)sizeof(T);
  while (V > 1 && (steps & (V - 1))) V >>= 1;
  if (A.interleaved && V < 2) return COMBO_EINVAL;  // (an odd stride: the caller copies)
  A.per_head = A.interleaved ? A.D / V : A.P / V + (A.D - 2 * A.P) / V;
  A.items = A.H * A.per_head;
  // tokens per workgroup: enough vectors for 256 threads x 4 where the tensor is large (>= 2048 workgroups left), one pass else
  const int cap = kTableBytes / (A.D * 4);
  long long T_ = A.tokens / 2048;
  const long long most = (1024 + A.items - 1) / A.items;
  if (T_ > most) T_ = most;
  if (T_ > cap) T_ = cap;
  if (T_ < 1) T_ = 1;
  A.T = (int)T_;
  if ((long long)A.T * A.items >= (1 << 16) && (A.T > 1 || A.items >= (1 << 24))) return COMBO_EINVAL;
  auto magic = [](unsigned d) { return d <= 1 ? 0u : (unsigned)((0x100000000ull + d - 1) / d); };
  A.items_magic = magic(A.items);
  A.head_magic = magic(A.per_head);
  const long long grid = (A.tokens + A.T - 1) / A.T;
  if (grid >= (1 << 24)) return COMBO_EINVAL;  // (a launch holds less than 2^32 threads)
  const size_t lds = (size_t)A.T * (A.D / 2) * sizeof(float2);
#define COMBO_GO(V_) hipLaunchKernelGGL((rotary_kernel<T, V_>), dim3((unsigned)grid), dim3(256), lds, st, A)
  switch (V) {
    case 8: if constexpr (sizeof(T) == 2) COMBO_GO(8); break;
    case 4: COMBO_GO(4); break;
    case 2: COMBO_GO(2); break;
    default: COMBO_GO(1);
  }
#undef COMBO_GO
  return (int)hipGetLastError();
}

}  // namespace

extern "C" int combo_rotary_axes(const void* x, long long stride_b, long long stride_n, long long stride_h, int dtype, const void* positions,
                                 int position_type, long long pos_stride_b, long long pos_stride_n, long long pos_stride_axis, int B, int N,
                                 int H, int D, int axes, const int* sections_host, const double* turns_host, int interleaved, int inverse,
                                 void* y, combo_stream_t stream) {
  if (!x || !positions || !y || !sections_host || !turns_host || B <= 0 || N <= 0 || H <= 0 || D <= 0 || (D & 1) || D > 2 * kMaxPairs ||
      axes <= 0 || axes > kMaxAxes || position_type < 0 || position_type > 3 || dtype < 0 || dtype > 2)
    return COMBO_EINVAL;
  RotaryArgs A;
  int P = 0;
  for (int a = 0; a < axes; ++a) {
    if (sections_host[a] < 0 || P + sections_host[a] > D / 2) return COMBO_EINVAL;
    for (int i = 0; i < sections_host[a]; ++i, ++P) {
      A.axis[P] = (unsigned char)a;
      A.turns[P] = turns_host[P];
    }
  }
  const int size = dtype == 0 ? 4 : 2;
  if (((uintptr_t)x | (uintptr_t)y) & (size - 1)) return COMBO_EINVAL;
  A.x = static_cast<const char*>(x);
  A.y = static_cast<char*>(y);
  A.pos = positions;
  A.xb = stride_b, A.xn = stride_n, A.xh = stride_h;
  A.pb = pos_stride_b, A.pn = pos_stride_n, A.pa = pos_stride_axis;
  A.tokens = (long long)B * N;
  A.N = N, A.H = H, A.D = D, A.P = P, A.interleaved = interleaved, A.inverse = inverse, A.pos_type = position_type;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) return launch<float>(A, st);
  if (dtype == 1) return launch<__bf16>(A, st);
  return launch<_Float16>(A, st);
}
