// rotary.hip — rotary embedding of query and key heads at given positions, in
// either pair layout, over the first R of D elements; alone, or behind the
// RMSNorm of each head, in one pass over q and k.
//
//   n = x * rsqrt(mean x^2 + eps) * w               (norm only)
//   pair (e, o), angle a of its position:  e' = e cos a - o sin a
//                                          o' = e sin a + o cos a
//   pairs: (2i, 2i + 1) interleaved, (i, i + R / 2) in halves; elements from R on
//   are copied.  In fp32, rounded once.
//   Backward of the norm: with d = R(-a) dy, n^ = x * r, g = d * w:
//     dx = r (g - n^ mean(g n^)),   dw = sum over rows of d n^
//   r is recomputed from x, which the backward reads anyway.
//
// Bound by reading and writing q and k once (x read again in the norm's backward).
// A group of LPR lanes holds a row, two 16-byte chunks per lane, R / 2 elements
// apart, so that a pair lies in one lane in either layout and a group's loads are
// contiguous.  A group takes U heads of one token with one load of the angles and
// with all rows in flight; they are spaced so that the groups of a wave take
// neighbouring heads at each step.  With U consecutive heads and the chunks of
// adjacent pairs side by side, the rotation below took 42 us, the norm 15 us.
//   rotation, bf16 B4 S2048 H32/8 D128 R64: 35.4 us, 4.7 TB/s (a copy: 5.1); U = 4 37, 1 34.4
//   rotation, fp32 B3 S1000 H12 D64:         7.7 us (U = 4: 8.7, 1: 9.2)
//   norm, fp16 B4 S4096 H32/8 D128: forward 65 us (U = 2: 64, 1: 70), backward 95 us
//   norm, bf16 B8 S1024 H12 D64: forward 11 us (U = 2: 14, 1: 13), backward 22 + 3.6 us
#include "mi_device.h"
#include "mi_kernels.h"

namespace mi {

namespace {

template <int DT>
struct Vec {
  static constexpr int N = DT == 0 ? 4 : 8;  // elements of 16 bytes
  typedef typename Store<DT>::type T;
  static __device__ __forceinline__ void unpack(u32x4 w, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == 0) {
        f[i] = __uint_as_float(w[i]);
      } else if constexpr (DT == 2) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        f[2 * i] = F16::to_f32((uint16_t)(w[i] & 0xffffu));
        f[2 * i + 1] = F16::to_f32((uint16_t)(w[i] >> 16));
      }
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float* f) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == 0) w[i] = __float_as_uint(f[i]);
      else if constexpr (DT == 2) w[i] = BF16::pack2(f[2 * i], f[2 * i + 1]);
      else w[i] = F16::pack2(f[2 * i], f[2 * i + 1]);
    }
    return w;
  }
};

__device__ __forceinline__ float load_as(int dt, const void* p, int64_t i) {
  if (dt == 0) return ((const float*)p)[i];
  const uint16_t x = ((const uint16_t*)p)[i];
  return dt == 2 ? bf16_to_f32(x) : f16_to_f32(x);
}

// N consecutive values of dtype dt (uniform), aligned to 16 bytes or to N values.
template <int N>
__device__ __forceinline__ void load_values(int dt, const void* p, int64_t i, float* f) {
  if (dt == 0) {
    if constexpr (N == 2) {
      const u32x2 w = *(const u32x2*)((const float*)p + i);
      f[0] = __uint_as_float(w[0]);
      f[1] = __uint_as_float(w[1]);
    }
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
      const f32x4 w = *(const f32x4*)((const float*)p + i + 4 * k);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * k + e] = w[e];
    }
  } else {
    uint32_t w[N / 2];
    if constexpr (N == 8) {
      const u32x4 x = *(const u32x4*)((const uint16_t*)p + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = x[k];
    } else if constexpr (N == 4) {
      const u32x2 x = *(const u32x2*)((const uint16_t*)p + i);
      w[0] = x[0];
      w[1] = x[1];
    } else {
      w[0] = *(const uint32_t*)((const uint16_t*)p + i);
    }
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
      if (dt == 2) {
        f[2 * k] = __uint_as_float(w[k] << 16);
        f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      } else {
        f[2 * k] = F16::to_f32((uint16_t)(w[k] & 0xffffu));
        f[2 * k + 1] = F16::to_f32((uint16_t)(w[k] >> 16));
      }
    }
  }
}

// Position of token (s, b); -1 if the tables do not have it.
__device__ __forceinline__ int64_t position(const RotaryArgs& a, int s, int b) {
  int64_t p = s;
  if (a.pos) {
    const int64_t i = s * a.pos_ss + b * a.pos_sb;
    p = a.pos64 ? ((const int64_t*)a.pos)[i] : ((const int*)a.pos)[i];
  }
  return p >= 0 && p < a.T ? p : -1;
}

// Sum over each aligned group of LPR lanes, the same bits in all of them.
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
  v = group_sum<(LPR < 8 ? LPR : 8)>(v);
  if constexpr (LPR >= 16) v = dpp_add<0x140>(v);  // row_mirror: the other 8 of 16 lanes
  if constexpr (LPR >= 32) v += __shfl_xor(v, 16, 64);
  return v;
}

enum { kRotate = 0, kNorm = 1, kNormGrad = 2 };

// Two chunks of pairs turned by the angles, in place.
template <int DT, int N>
__device__ __forceinline__ void turn(float (&f)[2 * N], const float (&cs)[N], const float (&sn)[N],
                                     bool interleaved, bool inverse) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float e = interleaved ? f[2 * i] : f[i], o = interleaved ? f[2 * i + 1] : f[N + i];
    float re, ro;
    rope_rotate<DT == 1>(e, o, cs[i], sn[i], inverse, re, ro);
    if (interleaved) {
      f[2 * i] = re;
      f[2 * i + 1] = ro;
    } else {
      f[i] = re;
      f[N + i] = ro;
    }
  }
}

// Where a lane's two chunks lie: pairs in the first R elements, then the rest.
struct Chunks {
  int c0, c1;
  bool have, turned;
};
template <int N>
__device__ __forceinline__ Chunks chunks(const RotaryArgs& a, int l) {
  const int half = a.R / (2 * N), lanes = a.D / (2 * N);  // lanes with pairs, all lanes
  Chunks c;
  c.have = l < lanes;
  c.turned = l < half;
  c.c0 = c.turned ? l : l + half;
  c.c1 = c.turned ? l + half : l + lanes;
  return c;
}

// The angles of a lane's pairs at position p (NaN where the tables end).
template <int N>
__device__ __forceinline__ void load_angles(const RotaryArgs& a, const Chunks& c, int64_t p,
                                            float (&cs)[N], float (&sn)[N]) {
  const int64_t row = p < 0 ? 0 : p;
  if (a.interleaved) {
    load_values<N / 2>(a.tab_dt, a.cos, row * a.cs_s + c.c0 * (N / 2), cs);
    load_values<N / 2>(a.tab_dt, a.cos, row * a.cs_s + c.c1 * (N / 2), cs + N / 2);
    load_values<N / 2>(a.tab_dt, a.sin, row * a.ss_s + c.c0 * (N / 2), sn);
    load_values<N / 2>(a.tab_dt, a.sin, row * a.ss_s + c.c1 * (N / 2), sn + N / 2);
  } else {
    load_values<N>(a.tab_dt, a.cos, row * a.cs_s + c.c0 * N, cs);
    load_values<N>(a.tab_dt, a.sin, row * a.ss_s + c.c0 * N, sn);
  }
  if (p < 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) cs[i] = sn[i] = __builtin_nanf("");
  }
}

template <int DT, int LPR, int MODE, int U>
__global__ __launch_bounds__(256) void rotary_vec_kernel(RotaryArgs a, FastDiv dhb, FastDiv dB,
                                                         uint32_t items) {
  constexpr int N = Vec<DT>::N;
  typedef typename Vec<DT>::T T;
  const uint32_t item = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (item >= items) return;  // whole groups
  const Chunks c = chunks<N>(a, threadIdx.x % LPR);
  // item = token * (head blocks of q and k) + head block
  const uint32_t sb = fdiv(item, dhb);
  int h0 = (int)(item - sb * dhb.d);
  const int qhb = (a.t[0].heads + U - 1) / U;
  const bool second = h0 >= qhb;
  if (second) h0 -= qhb;
  const RotaryTensor& t = a.t[second];
  const int dh = second ? (int)dhb.d - qhb : qhb;  // heads h0, h0 + dh, ...
  const uint32_t s = fdiv(sb, dB), b = sb - s * dB.d;
  const T* x = (const T*)t.x + s * t.x_ss + b * t.x_sb;
  T* out = (T*)t.out + s * t.o_ss + b * t.o_sb;

  u32x4 w[U][2];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    w[u][0] = w[u][1] = u32x4{0, 0, 0, 0};
    if (c.have && h0 + u * dh < t.heads) {
      w[u][0] = __builtin_nontemporal_load((const u32x4*)(x + (h0 + u * dh) * t.x_sh) + c.c0);
      w[u][1] = __builtin_nontemporal_load((const u32x4*)(x + (h0 + u * dh) * t.x_sh) + c.c1);
    }
  }
  float cs[N], sn[N];
  if (c.turned) load_angles<N>(a, c, position(a, s, b), cs, sn);
  float nw[2 * N];
  if (MODE == kNorm && c.have) {
    load_values<N>(a.w_dt, t.w, c.c0 * N, nw);
    load_values<N>(a.w_dt, t.w, c.c1 * N, nw + N);
  }
  const float inv_d = 1.f / a.D;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float f[2 * N];
    Vec<DT>::unpack(w[u][0], f);
    Vec<DT>::unpack(w[u][1], f + N);
    if constexpr (MODE == kNorm) {
      float q = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * N; ++i) q = __builtin_fmaf(f[i], f[i], q);
      const float r = rsqrtf(row_sum<LPR>(q) * inv_d + a.eps);
      if (c.have) {
#pragma unroll
        for (int i = 0; i < 2 * N; ++i) f[i] = f[i] * r * nw[i];
      }
    }
    if (!c.have || h0 + u * dh >= t.heads) continue;
    if (c.turned) turn<DT, N>(f, cs, sn, a.interleaved, MODE == kRotate && a.inverse);
    __builtin_nontemporal_store(Vec<DT>::pack(f), (u32x4*)(out + (h0 + u * dh) * t.o_sh) + c.c0);
    __builtin_nontemporal_store(Vec<DT>::pack(f + N), (u32x4*)(out + (h0 + u * dh) * t.o_sh) + c.c1);
  }
}

// Backward of norm and rotation.  Workgroups [0, a.blocks[0]) take q, the rest k;
// each sums dw over its rows and writes one partial row, added up in a fixed order
// by rotary_dw_kernel.
template <int DT, int LPR, int U>
__global__ __launch_bounds__(256) void rotary_grad_vec_kernel(RotaryArgs a, FastDiv dB) {
  constexpr int N = Vec<DT>::N, GROUPS = 256 / LPR;
  typedef typename Vec<DT>::T T;
  const int l = threadIdx.x % LPR;
  const Chunks c = chunks<N>(a, l);
  const bool second = (int)blockIdx.x >= a.blocks[0];
  const RotaryTensor& t = a.t[second];
  const uint32_t first = second ? blockIdx.x - a.blocks[0] : blockIdx.x;
  const uint32_t nhb = (t.heads + U - 1) / U, items = (uint32_t)a.S * a.B * nhb;
  float nw[2 * N], dw[2 * N];
#pragma unroll
  for (int i = 0; i < 2 * N; ++i) nw[i] = dw[i] = 0.f;
  if (c.have) {
    load_values<N>(a.w_dt, t.w, c.c0 * N, nw);
    load_values<N>(a.w_dt, t.w, c.c1 * N, nw + N);
  }
  const float inv_d = 1.f / a.D;
  for (uint32_t item = first * GROUPS + threadIdx.x / LPR; item < items;
       item += a.blocks[second] * GROUPS) {
    const uint32_t sb = item / nhb;
    const int h0 = item - sb * nhb;
    const uint32_t s = fdiv(sb, dB), b = sb - s * dB.d;
    const T* x = (const T*)t.x + s * t.x_ss + b * t.x_sb;
    const T* dy = (const T*)t.dy + s * t.dy_ss + b * t.dy_sb;
    T* out = (T*)t.out + s * t.o_ss + b * t.o_sb;
    u32x4 xw[U][2], dyw[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      xw[u][0] = xw[u][1] = dyw[u][0] = dyw[u][1] = u32x4{0, 0, 0, 0};
      if (c.have && h0 + u * (int)nhb < t.heads) {
        const int h = h0 + u * (int)nhb;
        xw[u][0] = __builtin_nontemporal_load((const u32x4*)(x + h * t.x_sh) + c.c0);
        xw[u][1] = __builtin_nontemporal_load((const u32x4*)(x + h * t.x_sh) + c.c1);
        dyw[u][0] = __builtin_nontemporal_load((const u32x4*)(dy + h * t.dy_sh) + c.c0);
        dyw[u][1] = __builtin_nontemporal_load((const u32x4*)(dy + h * t.dy_sh) + c.c1);
      }
    }
    float cs[N], sn[N];
    if (c.turned) load_angles<N>(a, c, position(a, s, b), cs, sn);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[2 * N], d[2 * N];
      Vec<DT>::unpack(xw[u][0], f);
      Vec<DT>::unpack(xw[u][1], f + N);
      Vec<DT>::unpack(dyw[u][0], d);
      Vec<DT>::unpack(dyw[u][1], d + N);
      if (c.turned) turn<0, N>(d, cs, sn, a.interleaved, true);
      float q = 0.f, gn = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * N; ++i) {
        q = __builtin_fmaf(f[i], f[i], q);
        gn = __builtin_fmaf(d[i] * nw[i], f[i], gn);
      }
      const float r = rsqrtf(row_sum<LPR>(q) * inv_d + a.eps);
      const float m = row_sum<LPR>(gn) * r * inv_d;  // mean(g n^)
      if (h0 + u * (int)nhb >= t.heads) continue;
#pragma unroll
      for (int i = 0; i < 2 * N; ++i) {
        const float n = f[i] * r;
        dw[i] = __builtin_fmaf(d[i], n, dw[i]);
        f[i] = r * (d[i] * nw[i] - n * m);
      }
      if (!c.have) continue;
      __builtin_nontemporal_store(Vec<DT>::pack(f), (u32x4*)(out + (h0 + u * (int)nhb) * t.o_sh) + c.c0);
      __builtin_nontemporal_store(Vec<DT>::pack(f + N), (u32x4*)(out + (h0 + u * (int)nhb) * t.o_sh) + c.c1);
    }
  }
  // groups of the wave, then the four waves
  __shared__ float sum[4][LPR * 2 * N];
#pragma unroll
  for (int i = 0; i < 2 * N; ++i) {
#pragma unroll
    for (int m = LPR; m < 64; m <<= 1) dw[i] += __shfl_xor(dw[i], m, 64);
    if ((threadIdx.x & 63) < LPR) sum[threadIdx.x >> 6][l * 2 * N + i] = dw[i];
  }
  __syncthreads();
  if (threadIdx.x < LPR && c.have) {
    float* p = a.part + (int64_t)blockIdx.x * a.D;
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
      const int at = l * 2 * N + i;
      p[(i < N ? c.c0 : c.c1) * N + i % N] = (sum[0][at] + sum[1][at]) + (sum[2][at] + sum[3][at]);
    }
  }
}

// One element of a row of any layout, turned: element i of D, as the vector path
// computes it.  ld(i): the row's value.
template <int DT, typename F>
__device__ __forceinline__ float turned(const RotaryArgs& a, int64_t p, int i, bool inverse, F ld) {
  const float x = ld(i);
  if (i >= a.R) return x;
  const int n = a.R / 2;
  const int k = a.interleaved ? i >> 1 : i < n ? i : i - n;
  const bool even = a.interleaved ? !(i & 1) : i < n;
  const int j = a.interleaved ? i ^ 1 : even ? i + n : i - n;
  float cs = __builtin_nanf(""), sn = cs;
  if (p >= 0) {
    cs = load_as(a.tab_dt, a.cos, p * a.cs_s + k * a.cs_i);
    sn = load_as(a.tab_dt, a.sin, p * a.ss_s + k * a.ss_i);
  }
  const float y = ld(j);
  float re, ro;
  rope_rotate<DT == 1>(even ? x : y, even ? y : x, cs, sn, inverse, re, ro);
  return even ? re : ro;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// Rows of any strides and sizes: a wave per row.  kNormGrad: D <= 512, workgroups
// as in rotary_grad_vec_kernel.
template <int DT, int MODE>
__global__ __launch_bounds__(256) void rotary_any_kernel(RotaryArgs a, uint32_t rows) {
  typedef typename Store<DT>::type T;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int NE = MODE == kNormGrad ? 8 : 1;
  float dw[NE] = {};
  const bool second = MODE == kNormGrad && (int)blockIdx.x >= a.blocks[0];
  uint32_t row = (second ? blockIdx.x - a.blocks[0] : blockIdx.x) * 4 + wave, step = 4 * gridDim.x;
  if (MODE == kNormGrad) {
    rows = (uint32_t)a.S * a.B * a.t[second].heads;
    step = 4 * a.blocks[second];
  }
  const int both = a.t[0].heads + a.t[1].heads;
  for (; row < rows; row += step) {
    const int nh = MODE == kNormGrad ? a.t[second].heads : both;
    const uint32_t sb = row / nh;
    int h = row - sb * nh;
    const uint32_t s = sb / a.B, b = sb - s * a.B;
    bool k = second;
    if (MODE != kNormGrad && h >= a.t[0].heads) {
      k = true;
      h -= a.t[0].heads;
    }
    const RotaryTensor& t = a.t[k];
    const T* x = (const T*)t.x + s * t.x_ss + b * t.x_sb + h * t.x_sh;
    T* out = (T*)t.out + s * t.o_ss + b * t.o_sb + h * t.o_sh;
    const int64_t p = position(a, s, b);
    float r = 1.f;
    if (MODE != kRotate) {
      float q = 0.f;
      for (int i = lane; i < a.D; i += 64) {
        const float v = Store<DT>::ld(x, i * t.x_sd);
        q = __builtin_fmaf(v, v, q);
      }
      r = rsqrtf(wave_sum(q) / a.D + a.eps);
    }
    if constexpr (MODE != kNormGrad) {
      auto ld = [&](int i) {
        float v = Store<DT>::ld(x, i * t.x_sd);
        if (MODE == kNorm) v = v * r * load_as(a.w_dt, t.w, i);
        return v;
      };
      for (int i0 = 0; i0 < a.D; i0 += 64) {
        const int i = i0 + lane;
        if (i < a.D) Store<DT>::st(out, i * t.o_sd, turned<DT>(a, p, i, a.inverse, ld));
      }
    } else {
      const T* dy = (const T*)t.dy + s * t.dy_ss + b * t.dy_sb + h * t.dy_sh;
      auto ld = [&](int i) { return Store<DT>::ld(dy, i * t.dy_sd); };
      float d[NE], n[NE], g[NE], gn = 0.f;
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const int i = lane + 64 * e;
        d[e] = n[e] = g[e] = 0.f;
        if (i < a.D) {
          d[e] = turned<0>(a, p, i, true, ld);
          n[e] = Store<DT>::ld(x, i * t.x_sd) * r;
          g[e] = d[e] * load_as(a.w_dt, t.w, i);
        }
        gn = __builtin_fmaf(g[e], n[e], gn);
      }
      const float m = wave_sum(gn) / a.D;
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const int i = lane + 64 * e;
        dw[e] = __builtin_fmaf(d[e], n[e], dw[e]);
        if (i < a.D) Store<DT>::st(out, i * t.o_sd, r * (g[e] - n[e] * m));
      }
    }
  }
  if constexpr (MODE == kNormGrad) {
    __shared__ float sum[4][512];
#pragma unroll
    for (int e = 0; e < NE; ++e) sum[wave][lane + 64 * e] = dw[e];
    __syncthreads();
    for (int i = threadIdx.x; i < a.D; i += 256)
      a.part[(int64_t)blockIdx.x * a.D + i] =
          (sum[0][i] + sum[1][i]) + (sum[2][i] + sum[3][i]);
  }
}

// dw of q (y = 0) and k (y = 1): the partial rows summed, 32 columns and 32 row
// lanes per workgroup.
__global__ __launch_bounds__(1024) void rotary_dw_kernel(RotaryArgs a) {
  __shared__ float sum[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x % 32, lane = threadIdx.x / 32;
  const int first = blockIdx.y ? a.blocks[0] : 0, n = a.blocks[blockIdx.y];
  float v = 0.f;
  if (col < a.D) {
#pragma unroll 8
    for (int i = lane; i < n; i += 32) v += a.part[(int64_t)(first + i) * a.D + col];
  }
  sum[lane][threadIdx.x % 32] = v;
  __syncthreads();
  if (lane == 0 && col < a.D) {
    v = 0.f;
    for (int i = 0; i < 32; ++i) v += sum[i][threadIdx.x];
    void* dw = a.t[blockIdx.y].dw;
    if (a.w_dt == 0) ((float*)dw)[col] = v;
    else ((uint16_t*)dw)[col] = a.w_dt == 2 ? f32_to_bf16(v) : f32_to_f16(v);
  }
}

template <int DT, int LPR>
hipError_t launch_vec(int mode, const RotaryArgs& a, hipStream_t st) {
  const FastDiv dB = make_fastdiv(a.B);
  if (mode == kNormGrad) {
    hipLaunchKernelGGL((rotary_grad_vec_kernel<DT, LPR, 2>), dim3(a.blocks[0] + a.blocks[1]),
                       dim3(256), 0, st, a, dB);
  } else {
    constexpr int UR = 2, U = 4;
    const int u = mode == kNorm ? U : UR;
    const uint32_t hb = (a.t[0].heads + u - 1) / u + (a.t[1].heads + u - 1) / u;
    const uint32_t items = (uint32_t)a.S * a.B * hb;
    const dim3 grid((items + 256 / LPR - 1) / (256 / LPR)), block(256);
    if (mode == kNorm)
      hipLaunchKernelGGL((rotary_vec_kernel<DT, LPR, kNorm, U>), grid, block, 0, st, a,
                         make_fastdiv(hb), dB, items);
    else
      hipLaunchKernelGGL((rotary_vec_kernel<DT, LPR, kRotate, UR>), grid, block, 0, st, a,
                         make_fastdiv(hb), dB, items);
  }
  return hipGetLastError();
}

template <int DT>
hipError_t launch_t(int mode, const RotaryArgs& a, bool vec, hipStream_t st) {
  if (vec) {
    const int lanes = a.D / (2 * Vec<DT>::N);
    if (lanes <= 4) return launch_vec<DT, 4>(mode, a, st);
    if (lanes <= 8) return launch_vec<DT, 8>(mode, a, st);
    if (lanes <= 16) return launch_vec<DT, 16>(mode, a, st);
    return launch_vec<DT, 32>(mode, a, st);
  }
  const uint32_t rows = (uint32_t)a.S * a.B * (a.t[0].heads + a.t[1].heads);
  const uint32_t wgs = rows / 4 + 1;  // they loop; a launch has at most 2^32 threads
  const dim3 grid(wgs < (1u << 22) ? wgs : 1u << 22), block(256);
  if (mode == kRotate)
    hipLaunchKernelGGL((rotary_any_kernel<DT, kRotate>), grid, block, 0, st, a, rows);
  else if (mode == kNorm)
    hipLaunchKernelGGL((rotary_any_kernel<DT, kNorm>), grid, block, 0, st, a, rows);
  else
    hipLaunchKernelGGL((rotary_any_kernel<DT, kNormGrad>), dim3(a.blocks[0] + a.blocks[1]), block,
                       0, st, a, rows);
  return hipGetLastError();
}

}  // namespace

// Workgroups of the norm's backward (partial rows of dw) for one tensor: at most
// 512, at least four rows to a wave.
int rotary_grad_blocks(int64_t rows) {
  const int64_t n = (rows + 15) / 16;
  return n > 512 ? 512 : (int)n;
}

// Row lengths that a group of at most 32 lanes holds, two whole chunks per lane,
// pairs in whole chunks.
bool rotary_vec_ok(int dtype, int D, int R) {
  const int n = dtype == 0 ? 4 : 8;
  return D % (2 * n) == 0 && R % (2 * n) == 0 && D / (2 * n) <= 32;
}

hipError_t launch_rotary(int dtype, int mode, const RotaryArgs& a, bool vec, hipStream_t st) {
  hipError_t e = dtype == 0   ? launch_t<0>(mode, a, vec, st)
                 : dtype == 1 ? launch_t<1>(mode, a, vec, st)
                              : launch_t<2>(mode, a, vec, st);
  if (e != hipSuccess || mode != kNormGrad) return e;
  hipLaunchKernelGGL(rotary_dw_kernel, dim3((a.D + 31) / 32, 2), dim3(1024), 0, st, a);
  return hipGetLastError();
}

}  // namespace mi
