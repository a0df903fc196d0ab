// Group norm with an activation on channels-last maps [B, HW, C] of fp32, bf16 or fp16, any channel count, forward and backward:
//     z = (x - mean[b, g]) rstd[b, g] w[c] + bias[c],  y = act(z),  act = none, ReLU, SiLU or GELU (erf)
//     dz = dy act'(z);  db[c] = sum dz;  dw[c] = sum dz xh;  dx = rstd (dz w - mean_g(dz w) - xh mean_g(dz w xh)),  xh = (x - mean) rstd
// The backward pass recomputes z from x: nothing but mean and rstd is kept, and the activation costs no tensor of its own.
//
// Bound: HBM.  A thread owns V neighbouring channels (16 bytes where the channel count and the pointers allow it) and walks the tokens, so
// per-channel constants stay in registers and all accesses are vectors, of as many values as divide the channel count (one, if that is odd).  Two shapes:
//   one launch   a workgroup owns one image and a few whole groups: it reads them for the statistics and again, out of the cache, for the
//                result.  For maps whose slice per workgroup is small (the launch then costs more than the traffic).
//   two launches partial statistics per (image, slice of tokens), then every workgroup of the second launch joins the partials of its own
//                image - a few KB out of L2 - and writes its tokens.
// 40 x 256 x 56 x 56 bf16 with SiLU (64 MB): forward 14 us for the statistics (4.6 TB/s) and 30 for the result (4.3), backward 32 for the sums (4.0)
// and 38 for dx (5.0), where a copy reaches 5.15; 3 x 60 x 117 x 93 fp16 with GELU (3.9 MB): 8, 9, 10 and 9 us; one 256 x 7 x 7 frame: 6.5 us.
// Statistics: a thread sums x - K and (x - K)^2 with K its own first value of the channel, in fp32, and hands on (mean, M2); these are
// joined as M2 = sum M2_i + sum n_i (mean_i - mean)^2.  K is one of the values, so the shift's cancellation is at most n_thread * 2^-24 of M2
// whatever the offset of the map (a plain sum of squares loses everything once mean^2 > 2^24 var).  All sums have a fixed order.
#include <initializer_list>

#include "combo_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxC = 4096;  // (a token's channel statistics and group results lie in 64 KiB of LDS)

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec { T v[V]; };

// 1 / x to one unit in the last place (v_rcp_f32): a full division is ten instructions, and a 16-bit activation map is short of them - SiLU by
// division took 39 us for a 64 MB bf16 map, half of it in the vector unit.  fp32 maps move twice the bytes and take the full functions.
__device__ __forceinline__ float quick_rcp(float x) { return __builtin_amdgcn_rcpf(x); }
template <bool FULL>
__device__ __forceinline__ float sigmoid(float z) {
  if constexpr (FULL) return 1.f / (1.f + expf(-z));
  return quick_rcp(1.f + __builtin_amdgcn_exp2f(-1.44269504f * z));
}

template <int N>
__device__ __forceinline__ float polynomial(const float (&c)[N], float x) {
  float y = c[N - 1];
#pragma unroll
  for (int i = N - 2; i >= 0; --i) y = fmaf(x, y, c[i]);
  return y;
}

// The normal distribution function and its density d(z).  With a = |z| the tail is R(a) exp(-a^2 / 2), and R, which falls from 1 / 2 like
// 1 / (a sqrt(2 pi)), is t (c0 + c1 t + ..) in t = 1 / (1 + s a) from a = 1 on, so the small side keeps its relative size; below that it is 1 / 2 + z P(z^2).
// Coefficients fitted here for the smallest relative error (weighted least squares): 7e-8 and 7e-10.  FULL: the exponent in two pieces (its rounding
// alone is 1.4e-6 of the value at z = -6) and a division, 7 u of either side, u = 2^-24; GELU over a normal z then has a root mean square error of 2.3e-8.
template <bool FULL>
__device__ __forceinline__ float normal_cdf(float z, float& density) {
  constexpr float kTail[7] = {0.11167358f, 0.11232360f, 0.09767063f, 0.10959552f, -0.0027825537f, 0.13058622f, -0.059144225f};
  constexpr float kCentre[6] = {0.39894229f, -0.06649036f, 0.009973324f, -0.0011863301f, 1.1348650e-4f, -7.6542565e-6f};
  const float a = fminf(fabsf(z), 15.f);  // (exp(-15^2 / 2) is 0 in fp32; a stays finite)
  const float h = a * a, x = -0.72134752f * h, u = fmaf(0.28f, a, 1.f);
  float e = __builtin_amdgcn_exp2f(x), t;
  if constexpr (FULL) {
    const float rest = fmaf(h, -0.72134752f, -x) + fmaf(h, -9.6298149e-9f, -0.72134752f * fmaf(a, a, -h));
    e = fmaf(0.69314718f * e, rest, e);
    t = 1.f / u;
  } else {
    t = quick_rcp(u);
  }
  density = 0.39894228f * e;
  const float tail = polynomial(kTail, t) * t * e;
  return a < 1.f ? fmaf(z, polynomial(kCentre, h), 0.5f) : z < 0.f ? tail : 1.f - tail;
}

// the same by one tail of six terms from a = 0 on, 4.6e-6 of it: 1 / 50 of half a step of fp16, for results that are rounded to 16 bits (forward, 40 x 256 x
// 56 x 56: 49.7 us, 53.4 with the function above).  Slopes do not take it: their sums, dw and db, come back in fp32 and were
// off by 3.5 u of their terms' sizes with it, 0.9 without.
__device__ __forceinline__ float normal_cdf_16(float z) {
  constexpr float kTail[6] = {0.12386069f, 0.12044134f, 0.13342951f, 0.015745264f, 0.18044983f, -0.073928952f};
  const float t = quick_rcp(fmaf(0.31f, fabsf(z), 1.f)), tail = polynomial(kTail, t) * t * __builtin_amdgcn_exp2f(-0.72134752f * z * z);
  return z < 0.f ? tail : 1.f - tail;
}

// FULL: to the last digits of fp32; else to what a 16-bit result shows of them
template <int ACT, bool FULL>
__device__ __forceinline__ float act(float z) {
  if constexpr (ACT == ACT_RELU) return z < 0.f ? 0.f : z;  // (a NaN stays one)
  if constexpr (ACT == ACT_SILU) return z * sigmoid<FULL>(z);
  if constexpr (ACT == ACT_GELU) {
    if constexpr (!FULL) return z * normal_cdf_16(z);
    float d;
    return z * normal_cdf<FULL>(z, d);
  }
  return z;
}
template <int ACT, bool FULL>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if constexpr (ACT == ACT_SILU) {
    const float s = sigmoid<FULL>(z);
    return s * fmaf(z, 1.f - s, 1.f);
  }
  if constexpr (ACT == ACT_GELU) {
    float d;
    const float c = normal_cdf<FULL>(z, d);
    return fmaf(z, d, c);
  }
  return 1.f;
}

struct NormArgs {
  const void *x, *dy;
  const float *w, *bias;      // nullable
  float *mean, *rstd;         // [B][G]
  float *part;                // forward: [B][S][G][2] (mean, M2); backward: [B][S][G][2] (s1, s2), then [B * S][C][2] (u, v)
  float *dw, *db;             // nullable
  void* out;
  float eps;
  int B, HW, C, G, per, S, slice;  // per: channels of a group; slice: tokens of a partial
  int range;                       // channels of a workgroup (the one-launch shape; else C)
};

// How a workgroup lies over [tokens][channels c0 .. c0 + range): a row of `width` threads covers the vectors of a token, `rows` such rows
// walk the tokens; a range of more than 256 vectors is walked in several sets.
struct Lanes {
  int width, rows, row, chunk;
  bool on;
  __device__ Lanes(int vectors) {
    width = min(vectors, kThreads);
    rows = kThreads / width;
    row = threadIdx.x / width;
    chunk = threadIdx.x - row * width;
    on = row < rows;
  }
};

__device__ __forceinline__ float team_sum(float v, int team) {
  for (int o = team >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// threads of a team that joins one group: a power of two <= 64 so that a team lies inside a wave
__device__ __forceinline__ int team_size(int groups) {
  int t = 64;
  while (t > 1 && kThreads / t < groups) t >>= 1;
  return t;
}

// (mean, M2) of `entries` (mean_i, M2_i, n_i): get(i, n, m, M2)
template <typename F>
__device__ __forceinline__ void join_stats(int entries, int team, int lane, F get, float& n, float& mean, float& M2) {
  float sn = 0.f, sm = 0.f;
  for (int i = lane; i < entries; i += team) {
    float ni, mi, qi;
    get(i, ni, mi, qi);
    sn += ni;
    sm += ni * mi;
  }
  n = team_sum(sn, team);
  mean = n > 0.f ? team_sum(sm, team) / n : 0.f;
  float q = 0.f;
  for (int i = lane; i < entries; i += team) {
    float ni, mi, qi;
    get(i, ni, mi, qi);
    if (ni > 0.f) q += qi + ni * (mi - mean) * (mi - mean);
  }
  M2 = team_sum(q, team);
}

// (mean, M2) of a token range into LDS: stat[rows][range / step][2], an entry for `step` neighbouring channels - V where a group is made of whole
// vectors, else 1
template <typename T, int V>
__device__ __forceinline__ void channel_stats(const T* x, int C, int range, int step, int t0, int t1, const Lanes& L, float* stat) {
  if (!L.on) return;
  for (int ch = L.chunk; ch * V < range; ch += kThreads) {
    const T* p = x + (long long)(t0 + L.row) * C + ch * V;
    float K[V], s[V], q[V];
#pragma unroll
    for (int k = 0; k < V; ++k) K[k] = s[k] = q[k] = 0.f;
    int n = 0;
    if (t0 + L.row < t1) {
      const Vec<T, V> a = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
      for (int k = 0; k < V; ++k) K[k] = (float)a.v[k];
      n = (t1 - t0 - L.row + L.rows - 1) / L.rows;
      const long long next = (long long)L.rows * C;
#pragma unroll 4
      for (int i = 1; i < n; ++i) {
        p += next;
        const Vec<T, V> b = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float d = (float)b.v[k] - K[k];
          s[k] += d;
          q[k] = fmaf(d, d, q[k]);
        }
      }
    }
    const float inv = n > 0 ? 1.f / (float)n : 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      q[k] -= s[k] * s[k] * inv;
      K[k] += s[k] * inv;
    }
    float* o = stat + (L.row * range + ch * V) / step * 2;
    if (step == 1) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        o[2 * k] = K[k];
        o[2 * k + 1] = q[k];
      }
    } else {
      float m = 0.f, M2 = 0.f;
#pragma unroll
      for (int k = 0; k < V; ++k) m += K[k];
      m *= 1.f / V;
#pragma unroll
      for (int k = 0; k < V; ++k) M2 += fmaf((K[k] - m) * (K[k] - m), (float)n, q[k]);
      o[0] = m;
      o[1] = M2;
    }
  }
}

// group g's statistics out of stat: a lane takes rows
__device__ __forceinline__ void group_of_stat(const float* stat, int range, int per, int step, int rows, int tokens, int g, int team, int lane,
                                              float& n, float& mean, float& M2) {
  const int width = range / step, q = per / step;
  const float* p = stat + 2 * g * q;
  float sn = 0.f, sm = 0.f;
  for (int r = lane; r < rows; r += team) {
    const float ni = r < tokens ? (float)((tokens - r + rows - 1) / rows) * step : 0.f;
    float m = 0.f;
    for (int c = 0; c < q; ++c) m += p[(r * width + c) * 2];
    sn += ni * q;
    sm += ni * m;
  }
  n = team_sum(sn, team);
  mean = n > 0.f ? team_sum(sm, team) / n : 0.f;
  float s2 = 0.f;
  for (int r = lane; r < rows; r += team) {
    if (r >= tokens) continue;
    const float ni = (float)((tokens - r + rows - 1) / rows) * step;
    for (int c = 0; c < q; ++c) {
      const float d = p[(r * width + c) * 2] - mean;
      s2 += fmaf(ni * d, d, p[(r * width + c) * 2 + 1]);
    }
  }
  M2 = team_sum(s2, team);
}

// partial statistics of one slice
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) gna_stats_kernel(const NormArgs A) {
  extern __shared__ float sh[];
  const int b = blockIdx.x / A.S, s = blockIdx.x - b * A.S;
  const int t0 = s * A.slice, t1 = min(A.HW, t0 + A.slice);
  const Lanes L(A.C / V);
  const int step = A.per % V == 0 ? V : 1;
  channel_stats<T, V>(static_cast<const T*>(A.x) + (long long)b * A.HW * A.C, A.C, A.C, step, t0, t1, L, sh);
  __syncthreads();
  const int team = team_size(A.G), lane = threadIdx.x & (team - 1);
  for (int g0 = 0; g0 < A.G; g0 += kThreads / team) {
    const int g = g0 + threadIdx.x / team;
    float n, mean, M2;
    group_of_stat(sh, A.C, A.per, step, L.rows, t1 - t0, min(g, A.G - 1), team, lane, n, mean, M2);
    if (lane == 0 && g < A.G) {
      float* o = A.part + (((long long)b * A.S + s) * A.G + g) * 2;
      o[0] = mean;
      o[1] = M2;
    }
  }
}

template <typename T, int V, int ACT>
__device__ __forceinline__ void apply_tokens(const NormArgs& A, int b, int c0, int range, int t0, int t1, const Lanes& L, const float* mean,
                                             const float* rstd) {
  if (!L.on) return;
  const T* x = static_cast<const T*>(A.x) + (long long)b * A.HW * A.C + c0;
  T* y = static_cast<T*>(A.out) + (long long)b * A.HW * A.C + c0;
  for (int ch = L.chunk; ch * V < range; ch += kThreads) {
    float m[V], a[V], bb[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = ch * V + k, g = c / A.per;
      m[k] = mean[g];
      a[k] = rstd[g] * (A.w ? A.w[c0 + c] : 1.f);
      bb[k] = A.bias ? A.bias[c0 + c] : 0.f;
    }
    long long off = (long long)(t0 + L.row) * A.C + ch * V;
    const long long step = (long long)L.rows * A.C;
#pragma unroll 4
    for (int t = t0 + L.row; t < t1; t += L.rows, off += step) {
      const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(x + off);
      Vec<T, V> o;
#pragma unroll
      for (int k = 0; k < V; ++k) o.v[k] = (T)act<ACT, sizeof(T) == 4>(fmaf((float)v.v[k] - m[k], a[k], bb[k]));
      *reinterpret_cast<Vec<T, V>*>(y + off) = o;
    }
  }
}

__device__ __forceinline__ float rstd_of(float M2, float n, float eps) { return 1.f / sqrtf(M2 / n + eps); }

// second launch: joins the partials of its image, normalises its slice
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads) gna_apply_kernel(const NormArgs A, int slice, int slices) {
  extern __shared__ float sh[];  // mean[G], rstd[G]
  const int b = blockIdx.x / slices, s = blockIdx.x - b * slices;
  const int team = team_size(A.G), lane = threadIdx.x & (team - 1);
  for (int g0 = 0; g0 < A.G; g0 += kThreads / team) {
    const int g = min(g0 + (int)threadIdx.x / team, A.G - 1);
    const float* part = A.part + ((long long)b * A.S * A.G + g) * 2;
    float n, mean, M2;
    join_stats(A.S, team, lane,
               [&](int i, float& ni, float& mi, float& qi) {
                 ni = (float)min(A.slice, A.HW - i * A.slice) * A.per;
                 mi = part[(long long)i * A.G * 2];
                 qi = part[(long long)i * A.G * 2 + 1];
               },
               n, mean, M2);
    if (lane == 0) {
      const float r = rstd_of(M2, n, A.eps);
      sh[g] = mean;
      sh[A.G + g] = r;
      if (s == 0 && A.mean) {
        A.mean[b * A.G + g] = mean;
        A.rstd[b * A.G + g] = r;
      }
    }
  }
  __syncthreads();
  const Lanes L(A.C / V);
  apply_tokens<T, V, ACT>(A, b, 0, A.C, s * slice, min(A.HW, (s + 1) * slice), L, sh, sh + A.G);
}

// one launch: an image's channels [c0, c0 + range) by one workgroup
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads) gna_forward_kernel(const NormArgs A) {
  extern __shared__ float sh[];
  const int parts = A.C / A.range, b = blockIdx.x / parts, c0 = (blockIdx.x - b * parts) * A.range;
  const int gn = A.range / A.per, g00 = c0 / A.per;
  const Lanes L(A.range / V);
  const int step = A.per % V == 0 ? V : 1;
  channel_stats<T, V>(static_cast<const T*>(A.x) + (long long)b * A.HW * A.C + c0, A.C, A.range, step, 0, A.HW, L, sh);
  __syncthreads();
  float* mr = sh + (size_t)L.rows * A.range * 2;
  const int team = team_size(gn), lane = threadIdx.x & (team - 1);
  for (int g0 = 0; g0 < gn; g0 += kThreads / team) {
    const int g = min(g0 + (int)threadIdx.x / team, gn - 1);
    float n, mean, M2;
    group_of_stat(sh, A.range, A.per, step, L.rows, A.HW, g, team, lane, n, mean, M2);
    if (lane == 0) {
      const float r = rstd_of(M2, n, A.eps);
      mr[g] = mean;
      mr[gn + g] = r;
      if (A.mean) {
        A.mean[b * A.G + g00 + g] = mean;
        A.rstd[b * A.G + g00 + g] = r;
      }
    }
  }
  __syncthreads();
  apply_tokens<T, V, ACT>(A, b, c0, A.range, 0, A.HW, L, mr, mr + gn);
}

// ---- backward ----

// per-channel (u, v) = (sum dz, sum dz xh) of a token range into LDS: uv[rows][range][2]
template <typename T, int V, int ACT>
__device__ __forceinline__ void channel_grads(const NormArgs& A, int b, int c0, int range, int t0, int t1, const Lanes& L, float* uv) {
  if (!L.on) return;
  const T* x = static_cast<const T*>(A.x) + (long long)b * A.HW * A.C + c0;
  const T* dy = static_cast<const T*>(A.dy) + (long long)b * A.HW * A.C + c0;
  for (int ch = L.chunk; ch * V < range; ch += kThreads) {
    float m[V], r[V], w[V], bb[V], u[V], v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = ch * V + k, g = b * A.G + (c0 + c) / A.per;
      m[k] = A.mean[g];
      r[k] = A.rstd[g];
      w[k] = A.w ? A.w[c0 + c] : 1.f;
      bb[k] = A.bias ? A.bias[c0 + c] : 0.f;
      u[k] = v[k] = 0.f;
    }
    long long off = (long long)(t0 + L.row) * A.C + ch * V;
    const long long step = (long long)L.rows * A.C;
#pragma unroll 2
    for (int t = t0 + L.row; t < t1; t += L.rows, off += step) {
      const Vec<T, V> xv = *reinterpret_cast<const Vec<T, V>*>(x + off), gv = *reinterpret_cast<const Vec<T, V>*>(dy + off);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float xh = ((float)xv.v[k] - m[k]) * r[k];
        const float dz = (float)gv.v[k] * act_slope<ACT, sizeof(T) == 4>(fmaf(xh, w[k], bb[k]));
        u[k] += dz;
        v[k] = fmaf(dz, xh, v[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float* o = uv + (L.row * range + ch * V + k) * 2;
      o[0] = u[k];
      o[1] = v[k];
    }
  }
}

// joins the rows of uv[rows][range][2] into row 0, writes them to `chan` [range][2] and the group sums (sum_c w u, sum_c w v) to s12[gn][2]
__device__ __forceinline__ void join_grads(const NormArgs& A, int c0, int range, const Lanes& L, float* uv, float* chan, float* s12) {
  for (int i = threadIdx.x; i < range; i += kThreads) {
    float u = 0.f, v = 0.f;
    for (int r = 0; r < L.rows; ++r) {
      u += uv[(r * range + i) * 2];
      v += uv[(r * range + i) * 2 + 1];
    }
    chan[2 * i] = u;
    chan[2 * i + 1] = v;
    const float w = A.w ? A.w[c0 + i] : 1.f;
    uv[2 * i] = u * w;
    uv[2 * i + 1] = v * w;
  }
  __syncthreads();
  const int gn = range / A.per, team = team_size(gn), lane = threadIdx.x & (team - 1);
  for (int g0 = 0; g0 < gn; g0 += kThreads / team) {
    const int g = min(g0 + (int)threadIdx.x / team, gn - 1);
    float a = 0.f, q = 0.f;
    for (int c = lane; c < A.per; c += team) {
      a += uv[(g * A.per + c) * 2];
      q += uv[(g * A.per + c) * 2 + 1];
    }
    a = team_sum(a, team);
    q = team_sum(q, team);
    if (lane == 0) {
      s12[2 * g] = a;
      s12[2 * g + 1] = q;
    }
  }
}

// s12: [gn][2] of this image's groups from c0 on
template <typename T, int V, int ACT>
__device__ __forceinline__ void dx_tokens(const NormArgs& A, int b, int c0, int range, int t0, int t1, const Lanes& L, const float* s12) {
  if (!L.on) return;
  const long long base = (long long)b * A.HW * A.C + c0;
  const T* x = static_cast<const T*>(A.x) + base;
  const T* dy = static_cast<const T*>(A.dy) + base;
  T* dx = static_cast<T*>(A.out) + base;
  const float inv_n = 1.f / ((float)A.HW * (float)A.per);
  for (int ch = L.chunk; ch * V < range; ch += kThreads) {
    float m[V], r[V], w[V], bb[V], a1[V], a2[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = ch * V + k, gl = c / A.per, g = b * A.G + c0 / A.per + gl;
      m[k] = A.mean[g];
      r[k] = A.rstd[g];
      w[k] = A.w ? A.w[c0 + c] : 1.f;
      bb[k] = A.bias ? A.bias[c0 + c] : 0.f;
      a1[k] = s12[2 * gl] * inv_n;
      a2[k] = s12[2 * gl + 1] * inv_n;
    }
    long long off = (long long)(t0 + L.row) * A.C + ch * V;
    const long long step = (long long)L.rows * A.C;
#pragma unroll 2
    for (int t = t0 + L.row; t < t1; t += L.rows, off += step) {
      const Vec<T, V> xv = *reinterpret_cast<const Vec<T, V>*>(x + off), gv = *reinterpret_cast<const Vec<T, V>*>(dy + off);
      Vec<T, V> o;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float xh = ((float)xv.v[k] - m[k]) * r[k];
        const float dz = (float)gv.v[k] * act_slope<ACT, sizeof(T) == 4>(fmaf(xh, w[k], bb[k]));
        o.v[k] = (T)(r[k] * fmaf(-xh, a2[k], fmaf(dz, w[k], -a1[k])));
      }
      *reinterpret_cast<Vec<T, V>*>(dx + off) = o;
    }
  }
}

__device__ __forceinline__ float* chan_of(const NormArgs& A) { return A.part + (long long)A.B * A.S * A.G * 2; }

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads) gna_grad_partial_kernel(const NormArgs A) {
  extern __shared__ float sh[];
  const int b = blockIdx.x / A.S, s = blockIdx.x - b * A.S;
  const Lanes L(A.C / V);
  channel_grads<T, V, ACT>(A, b, 0, A.C, s * A.slice, min(A.HW, (s + 1) * A.slice), L, sh);
  __syncthreads();
  join_grads(A, 0, A.C, L, sh, chan_of(A) + (long long)blockIdx.x * A.C * 2, A.part + (long long)blockIdx.x * A.G * 2);
}

// dw, db: 16 channels by 16 rows of partials per workgroup, joined in a fixed order
__device__ __forceinline__ void param_grads(const NormArgs& A, int block, int rows_total, float* sh) {
  const int c = block * 16 + (threadIdx.x & 15), r0 = threadIdx.x >> 4;
  const float* p = chan_of(A);
  float u = 0.f, v = 0.f;
  if (c < A.C) {
#pragma unroll 4
    for (int r = r0; r < rows_total; r += 16) {
      const float2 a = *reinterpret_cast<const float2*>(p + ((long long)r * A.C + c) * 2);
      u += a.x;
      v += a.y;
    }
  }
  sh[threadIdx.x] = u;
  sh[256 + threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.x < 16 && c < A.C) {
    for (int r = 1; r < 16; ++r) {
      u += sh[r * 16 + threadIdx.x];
      v += sh[256 + r * 16 + threadIdx.x];
    }
    if (A.dw) A.dw[c] = v;
    if (A.db) A.db[c] = u;
  }
}

// second launch: the first workgroups join dw and db, the others write dx
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads) gna_grad_apply_kernel(const NormArgs A, int slice, int slices, int param_blocks) {
  extern __shared__ float sh[];
  if ((int)blockIdx.x < param_blocks) {
    param_grads(A, blockIdx.x, A.B * A.S, sh);
    return;
  }
  const int id = blockIdx.x - param_blocks, b = id / slices, s = id - b * slices;
  const int team = team_size(A.G), lane = threadIdx.x & (team - 1);
  for (int g0 = 0; g0 < A.G; g0 += kThreads / team) {
    const int g = min(g0 + (int)threadIdx.x / team, A.G - 1);
    float a = 0.f, q = 0.f;
    for (int i = lane; i < A.S; i += team) {
      const float* p = A.part + (((long long)b * A.S + i) * A.G + g) * 2;
      a += p[0];
      q += p[1];
    }
    a = team_sum(a, team);
    q = team_sum(q, team);
    if (lane == 0) {
      sh[2 * g] = a;
      sh[2 * g + 1] = q;
    }
  }
  __syncthreads();
  const Lanes L(A.C / V);
  dx_tokens<T, V, ACT>(A, b, 0, A.C, s * slice, min(A.HW, (s + 1) * slice), L, sh);
}

// one launch for dx (S = 1: the channel sums of an image are one row of partials); dw and db follow in gna_param_kernel
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads) gna_backward_kernel(const NormArgs A) {
  extern __shared__ float sh[];
  const int parts = A.C / A.range, b = blockIdx.x / parts, c0 = (blockIdx.x - b * parts) * A.range;
  const Lanes L(A.range / V);
  float* s12 = sh + (size_t)L.rows * A.range * 2;
  channel_grads<T, V, ACT>(A, b, c0, A.range, 0, A.HW, L, sh);
  __syncthreads();
  join_grads(A, c0, A.range, L, sh, chan_of(A) + ((long long)b * A.C + c0) * 2, s12);
  __syncthreads();
  dx_tokens<T, V, ACT>(A, b, c0, A.range, 0, A.HW, L, s12);
}

__global__ void __launch_bounds__(kThreads) gna_param_kernel(const NormArgs A) {
  __shared__ float sh[512];
  param_grads(A, blockIdx.x, A.B, sh);
}

// ---- host ----

// channels of a workgroup in the one-launch shape: the fewest whole groups that make whole vectors and at least a cache line
int channel_range(int C, int G, int V, int size) {
  const int per = C / G;
  for (int k = 1; k < G; ++k)
    if (G % k == 0 && (k * per) % V == 0 && k * per * size >= 128) return k * per;
  return C;
}

int vector_of(int C, int size, uintptr_t all) {
  int V = 16 / size;
  while (V > 1 && (C % V || all % (V * size))) V >>= 1;
  return V;
}

// One launch while a workgroup's slice is at most 128 KiB, i.e. at most ~4 us of one CU's cache traffic, less than a second launch and
// its join cost; a large map goes over the whole chip in two.
bool one_launch(const NormArgs& A, int size) { return (long long)A.HW * A.range * size <= 131072; }

size_t lds_floats(int range, int V) {
  const int vectors = range / V, rows = vectors < kThreads ? kThreads / vectors : 1;
  return (size_t)rows * range * 2;
}

// slices of an image: the batch makes just under 1024 workgroups, four for each CU (40 images in 26 slices were 1040, and the CUs with five
// of them finished last: 39 us against 31), with at least 16 tokens and 8 KiB in each.  At most 256 an image, one a CU where there is but one: every
// workgroup of the second launch joins all partials of its image, and with up to 1024 of them 1 x 256 x 112 x 112 bf16 takes 85 us forward and 155 in
// training, with 256 27 and 53 (1 x 256 x 512 x 512, which has the work for it: 159 and 357 against 128 and 447)
void choose_slices(NormArgs& A, int size) {
  long long by_bytes = ((long long)A.HW * A.C * size + 8191) / 8192;
  long long want = 1024 / A.B;
  long long S = by_bytes < want ? by_bytes : want;
  if (S > (A.HW + 15) / 16) S = (A.HW + 15) / 16;
  if (S > 256) S = 256;
  if (S < 1) S = 1;
  A.slice = (int)((A.HW + S - 1) / S);
  A.S = (A.HW + A.slice - 1) / A.slice;
}

template <typename T, int V, int ACT>
int forward(NormArgs& A, hipStream_t st) {
  if (one_launch(A, sizeof(T))) {
    const size_t lds = (lds_floats(A.range, V) + 2 * (A.range / A.per)) * sizeof(float);
    hipLaunchKernelGGL((gna_forward_kernel<T, V, ACT>), dim3(A.B * (A.C / A.range)), dim3(kThreads), lds, st, A);
    return (int)hipGetLastError();
  }
  hipLaunchKernelGGL((gna_stats_kernel<T, V>), dim3(A.B * A.S), dim3(kThreads), lds_floats(A.C, V) * sizeof(float), st, A);
  hipLaunchKernelGGL((gna_apply_kernel<T, V, ACT>), dim3(A.B * A.S), dim3(kThreads), (size_t)A.G * 2 * sizeof(float), st, A, A.slice, A.S);
  return (int)hipGetLastError();
}

template <typename T, int V, int ACT>
int backward(NormArgs& A, hipStream_t st) {
  const int param_blocks = A.dw || A.db ? (A.C + 15) / 16 : 0;
  if (one_launch(A, sizeof(T))) {
    A.S = 1;
    const size_t lds = (lds_floats(A.range, V) + 2 * (A.range / A.per)) * sizeof(float);
    hipLaunchKernelGGL((gna_backward_kernel<T, V, ACT>), dim3(A.B * (A.C / A.range)), dim3(kThreads), lds, st, A);
    if (param_blocks) hipLaunchKernelGGL(gna_param_kernel, dim3(param_blocks), dim3(kThreads), 0, st, A);
    return (int)hipGetLastError();
  }
  hipLaunchKernelGGL((gna_grad_partial_kernel<T, V, ACT>), dim3(A.B * A.S), dim3(kThreads), lds_floats(A.C, V) * sizeof(float), st, A);
  const size_t lds = (size_t)(A.G * 2 > 512 ? A.G * 2 : 512) * sizeof(float);
  hipLaunchKernelGGL((gna_grad_apply_kernel<T, V, ACT>), dim3(param_blocks + A.B * A.S), dim3(kThreads), lds, st, A, A.slice, A.S, param_blocks);
  return (int)hipGetLastError();
}

template <typename T, int V>
int by_act(NormArgs& A, int act_, bool back, hipStream_t st) {
  switch (act_) {
    case ACT_NONE: return back ? backward<T, V, ACT_NONE>(A, st) : forward<T, V, ACT_NONE>(A, st);
    case ACT_RELU: return back ? backward<T, V, ACT_RELU>(A, st) : forward<T, V, ACT_RELU>(A, st);
    case ACT_SILU: return back ? backward<T, V, ACT_SILU>(A, st) : forward<T, V, ACT_SILU>(A, st);
    default: return back ? backward<T, V, ACT_GELU>(A, st) : forward<T, V, ACT_GELU>(A, st);
  }
}

template <typename T>
int by_width(NormArgs& A, int act_, bool back, uintptr_t all, hipStream_t st) {
  const int V = vector_of(A.C, sizeof(T), all);
  A.range = channel_range(A.C, A.G, V, sizeof(T));
  choose_slices(A, sizeof(T));
  switch (V) {
    case 8: if constexpr (sizeof(T) == 2) return by_act<T, 8>(A, act_, back, st); break;
    case 4: return by_act<T, 4>(A, act_, back, st);
    case 2: return by_act<T, 2>(A, act_, back, st);
    default: return by_act<T, 1>(A, act_, back, st);
  }
  return COMBO_EINVAL;
}

int run(NormArgs& A, int dtype, int act_, bool back, uintptr_t all, hipStream_t st) {
  if (dtype == 0) return by_width<float>(A, act_, back, all, st);
  if (dtype == 1) return by_width<__bf16>(A, act_, back, all, st);
  return by_width<_Float16>(A, act_, back, all, st);
}

// (B * lines bounds every grid: a launch holds less than 2^32 threads)
bool shape_ok(int B, int HW, int C, int G, int dtype, int act_) {
  if (B <= 0 || HW <= 0 || HW > (1 << 30) || C <= 0 || C > kMaxC || G <= 0 || C % G || dtype < 0 || dtype > 2 || act_ < 0 || act_ > 3) return false;
  const int lines = (C * (dtype == 0 ? 4 : 2) + 127) / 128;
  return (long long)B * C < 0x7fffffffll && B <= (1 << 22) && (long long)B * lines < (1 << 24);
}

bool floats_ok(std::initializer_list<const float*> all, const float* workspace) {
  uintptr_t a = 0;
  for (const float* p : all) a |= (uintptr_t)p;
  return !(a & 3) && !((uintptr_t)workspace & 7);  // (the workspace is read in pairs)
}

}  // namespace

extern "C" {

long long combo_groupnorm_act_workspace(int B, int HW, int C, int G, int dtype, int backward_pass) {
  if (!shape_ok(B, HW, C, G, dtype, 0)) return -1;
  NormArgs A = {};
  A.B = B, A.HW = HW, A.C = C, A.G = G, A.range = C;
  if (!backward_pass && one_launch(A, dtype == 0 ? 4 : 2)) return 0;
  choose_slices(A, dtype == 0 ? 4 : 2);
  const long long rows = (long long)B * A.S;
  return rows * G * 2 + (backward_pass ? rows * C * 2 : 0);
}

int combo_groupnorm_act_forward(const void* x, const float* weight, const float* bias, int B, int HW, int C, int G, float eps, int act_,
                                int dtype, float* workspace, float* mean, float* rstd, void* y, combo_stream_t stream) {
  if (!x || (!mean) != (!rstd) || !y || !shape_ok(B, HW, C, G, dtype, act_)) return COMBO_EINVAL;
  if (!workspace && combo_groupnorm_act_workspace(B, HW, C, G, dtype, 0) > 0) return COMBO_EINVAL;
  const uintptr_t all = (uintptr_t)x | (uintptr_t)y;
  if (all & (dtype == 0 ? 3 : 1) || !floats_ok({weight, bias, mean, rstd}, workspace)) return COMBO_EINVAL;
  NormArgs A = {};
  A.x = x, A.w = weight, A.bias = bias, A.mean = mean, A.rstd = rstd, A.part = workspace, A.out = y, A.eps = eps;
  A.B = B, A.HW = HW, A.C = C, A.G = G, A.per = C / G;
  return run(A, dtype, act_, false, all, (hipStream_t)stream);
}

int combo_groupnorm_act_backward(const void* dy, const void* x, const float* weight, const float* bias, const float* mean, const float* rstd,
                                 int B, int HW, int C, int G, int act_, int dtype, float* workspace, void* dx, float* dweight, float* dbias,
                                 combo_stream_t stream) {
  if (!dy || !x || !mean || !rstd || !workspace || !dx || !shape_ok(B, HW, C, G, dtype, act_)) return COMBO_EINVAL;
  const uintptr_t all = (uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx;
  if (all & (dtype == 0 ? 3 : 1) || !floats_ok({weight, bias, mean, rstd, dweight, dbias}, workspace)) return COMBO_EINVAL;
  NormArgs A = {};
  A.x = x, A.dy = dy, A.w = weight, A.bias = bias, A.mean = const_cast<float*>(mean), A.rstd = const_cast<float*>(rstd), A.part = workspace;
  A.out = dx, A.dw = dweight, A.db = dbias;
  A.B = B, A.HW = HW, A.C = C, A.G = G, A.per = C / G;
  return run(A, dtype, act_, true, all, (hipStream_t)stream);
}

}  // extern "C"
