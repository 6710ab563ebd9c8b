// decode.hip — attention of one new token of each sequence over its cache, with
// the forward's score modifications (sattn_device.h): the query is the last of
// the sequence's len keys.
//
// Bound by reading the cache once: 2 * len * Hk * D elements against 4 * H * D
// operations per key.  The query heads that share a key head are the columns of
// one matrix-core operand (up to 32 of them, the rest of the columns idle), so
// the cache is read once for all of them, and the products stay far below the
// memory time whatever the group.  B32 H32/8 D128, lengths 512 to 4096: 57 us for 337 MB
// (5.9 TB/s); B1 H16/4 S65536 with a cap: 26 us for 134 MB (5.2 TB/s); joins 5 us each.
//   * A workgroup takes one key head of one sequence and one of `splits` equal
//     parts of its keys; its waves take 32-key blocks of the tiles that all of
//     them stage (global -> LDS, double buffered), and merge at the end.
//   * With more than one part, each writes its O (unnormalised), maximum and sum
//     to the workspace, and a second launch joins them.  Rows at or past len are
//     never read.
#include <type_traits>

#include "sattn_device.h"

namespace mi {

namespace {

// Waves per workgroup: two, so that two workgroups share a CU (64 KB of tiles each at
// D = 128; one for fp32) and one streams while the other starts or merges.  Four
// (one workgroup per CU): 71 against 65 us at B32 H32/8 S <= 4096, lengths of 1/8 to 1.
template <typename E, int D>
constexpr int kWaves = 2;
constexpr int kMaxParts = 64;  // B1 H16/4 S65536: 31 us; 128 the same, 256 43

template <typename E>
__device__ __forceinline__ void put(void* p, int64_t i, float x) {
  if constexpr (Elem<E>::kBytes == 4)
    ((float*)p)[i] = x;
  else
    ((uint16_t*)p)[i] = (uint16_t)(E::pack2(x, 0.f) & 0xffffu);
}

template <typename E, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__((64 * kWaves<E, D>), 1) void decode_kernel(DecodeArgs a) {
  using L = Lay<E, D>;
  constexpr int NW = kWaves<E, D>, TK = 32 * NW;
  __shared__ __attribute__((aligned(16))) char K0[TK * L::RB];
  __shared__ __attribute__((aligned(16))) char K1[TK * L::RB];
  __shared__ __attribute__((aligned(16))) char V0[TK * L::RB];
  __shared__ __attribute__((aligned(16))) char V1[TK * L::RB];
  __shared__ float ML[2][NW][32];

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // blockIdx.x: sequence, block of 32 heads of a group, key head (fastest); y: part
  const int nhb = (a.G + 31) / 32;
  const int hk = blockIdx.x % a.Hk, hb = blockIdx.x / a.Hk % nhb, b = blockIdx.x / (a.Hk * nhb);
  const int h0 = hk * a.G + 32 * hb, nh = min(32, a.G - 32 * hb);
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.S) : a.S;
  const int nt = (len + TK - 1) / TK;
  const int t0 = (int)((int64_t)nt * blockIdx.y / a.splits);
  const int t1 = (int)((int64_t)nt * (blockIdx.y + 1) / a.splits);

  const char* qp = (const char*)a.q + (b * a.q_sb + (h0 + l32) * a.q_sh) * L::ESZ;
  u32x4 qf[L::KS];
#pragma unroll
  for (int ks = 0; ks < L::KS; ++ks)
    qf[ks] = l32 < nh && 2 * ks + g < a.dch ? *(const u32x4*)(qp + 16 * (2 * ks + g))
                                             : u32x4{0, 0, 0, 0};
  const float slope2 = BIAS && l32 < nh ? a.slopes[h0 + l32] * kLog2e : 0.f;

  // read once: non-temporal (72 against 77 us at the size above)
  Stage<E, D, TK, NW, kOnce> ksrc, vsrc;
  ksrc.init(a.k, b, hk, a.dch, lane, wave);
  vsrc.init(a.v, b, hk, a.dch, lane, wave);
  Reads<E, D> rd;
  rd.init(lane);

  f32x16 acc[L::DB];
#pragma unroll
  for (int i = 0; i < L::DB; ++i) acc[i] = f32x16{};
  float m_run = -INFINITY, l_run = 0.f;
  if (t0 < t1) {
    ksrc.load(t0 * TK, len, K0, wave);
    vsrc.load(t0 * TK, len, V0, wave);
    __syncthreads();
  }
  auto step = [&](int t, auto slot) __attribute__((always_inline)) {
    constexpr int I = decltype(slot)::value;
    const char* kt = (I ? K1 : K0) + 32 * wave * L::RB;
    const char* vt = (I ? V1 : V0) + 32 * wave * L::RB;
    if (t + 1 < t1) {
      ksrc.load((t + 1) * TK, len, I ? K0 : K1, wave);
      vsrc.load((t + 1) * TK, len, I ? V0 : V1, wave);
    }
    rd.refresh();
    const int k0 = t * TK + 32 * wave;
    if (k0 < len) {
      f32x16 s;
#pragma unroll
      for (int ks = 0; ks < L::KS; ++ks)
        s = Elem<E>::mfma(rd.row(kt, 0, ks), qf[ks], ks == 0 ? f32x16{} : s);
      const float d0 = (float)(len - 1 - k0 - 4 * g);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = score_y<E, CAP>(s[r], a.sc) * a.sc.f;
        // no key is behind the query's position, which is the last
        if constexpr (BIAS) s[r] = __builtin_fmaf(-slope2, d0 - (8 * (r >> 2) + (r & 3)), s[r]);
      }
      if (k0 + 32 > len) {
        const int rel = len - k0 - 4 * g;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (8 * (r >> 2) + (r & 3) >= rel) s[r] = -INFINITY;
      }
      float mx = vmax(s[0], s[1]);
#pragma unroll
      for (int r = 2; r < 16; r += 2) mx = vmax(vmax(mx, s[r]), s[r + 1]);
      mx = max_halves(mx);
      if (__any(mx > m_run)) {
        const float m_new = fmaxf(m_run, mx);
        const float alpha = fast_exp2(m_run - (m_new == -INFINITY ? 0.f : m_new));
        l_run *= alpha;
#pragma unroll
        for (int db = 0; db < L::DB; ++db) acc[db] *= alpha;
        m_run = m_new;
      }
      const float ref = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = fast_exp2(s[r] - ref);
#pragma unroll
      for (int ng = 0; ng < L::NG; ++ng) {
        const u32x4 p = Elem<E>::operand(s, ng);
        l_run = Elem<E>::sum(p, l_run);
#pragma unroll
        for (int db = 0; db < L::DB; ++db)
          acc[db] = Elem<E>::mfma(rd.col(vt, 0, ng, db), p, acc[db]);
      }
    }
    __syncthreads();
  };
  int t = t0;
  for (; t + 1 < t1; t += 2) {
    step(t, std::integral_constant<int, 0>{});
    step(t + 1, std::integral_constant<int, 1>{});
  }
  if (t < t1) step(t, std::integral_constant<int, 0>{});

  // Merge the waves: each takes its sums to the common maximum and leaves its
  // O^T, as [head][D] floats, in a tile buffer (idle, and large enough); element d of
  // head h sits at d ^ h, so that neither side meets in a bank.
  const float l = sum_halves(l_run);
  if (g == 0) {
    ML[0][wave][l32] = m_run;
    ML[1][wave][l32] = l;
  }
  __syncthreads();
  float m = ML[0][0][l32], lt = 0.f;
#pragma unroll
  for (int w = 1; w < NW; ++w) m = fmaxf(m, ML[0][w][l32]);
  const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int w = 0; w < NW; ++w) lt += ML[1][w][l32] * fast_exp2(ML[0][w][l32] - ref);
  const float f = fast_exp2(m_run - ref);
  // one part: normalised here
  const float fo = a.splits == 1 ? (lt == 0.f ? 0.f : f / lt) : f;
  float* const mine = (float*)(wave == 0 ? K0 : K1);
  static_assert(NW == 2 && TK * L::RB >= 32 * D * 4, "merge buffers");
#pragma unroll
  for (int db = 0; db < L::DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      mine[l32 * D + ((32 * db + 8 * (r >> 2) + 4 * g + (r & 3)) ^ l32)] = acc[db][r] * fo;
  __syncthreads();
  const int64_t row0 = (int64_t)b * a.H + h0;
  for (int i = tid; i < nh * D; i += 64 * NW) {
    const int hh = i / D, d = i % D, at = hh * D + (d ^ hh);
    if (d >= a.D) continue;
    const float x = ((float*)K0)[at] + ((float*)K1)[at];
    if (a.splits == 1)
      put<E>(a.o, b * a.o_sb + (h0 + hh) * a.o_sh + d, x);
    else
      a.part[((row0 + hh) * a.splits + blockIdx.y) * a.D + d] = x;
  }
  if (a.splits > 1 && tid < nh) {
    float* ml = a.ml + 2 * ((row0 + tid) * a.splits + blockIdx.y);
    ml[0] = m;
    ml[1] = lt;
  }
}

// O of one row from its parts: a workgroup of JW waves per row, lane d, d + 64.  The
// time is each wave's chain of loads (one wave over 64 parts took 35 us), kept to four
// parts, all in flight: 16 waves, or 4 for up to 16 parts, where many rows would only
// start waves (B32 H32: 68 against 65 us).
template <typename E, int JW>
__global__ __launch_bounds__(64 * JW) void decode_join_kernel(DecodeArgs a) {
  __shared__ float sum[JW][128], weight[kMaxParts];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const float* ml = a.ml + 2 * row * a.splits;
  float mt = -INFINITY;
  for (int i = lane; i < a.splits; i += 64) mt = fmaxf(mt, ml[2 * i]);
#pragma unroll
  for (int x = 32; x; x >>= 1) mt = fmaxf(mt, __shfl_xor(mt, x, 64));
  float lt = 0.f;
  for (int i = lane; i < a.splits; i += 64) {
    const float f = fast_exp2(ml[2 * i] - (mt == -INFINITY ? 0.f : mt));
    lt = __builtin_fmaf(ml[2 * i + 1], f, lt);
    if (wave == 0) weight[i] = f;
  }
#pragma unroll
  for (int x = 32; x; x >>= 1) lt += __shfl_xor(lt, x, 64);
  __syncthreads();
  const float* part = a.part + row * a.splits * a.D;
  float o0 = 0.f, o1 = 0.f;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int s = wave + JW * n;
    if (s >= a.splits) break;
    const float w = weight[s];
    if (lane < a.D) o0 = __builtin_fmaf(part[s * a.D + lane], w, o0);
    if (lane + 64 < a.D) o1 = __builtin_fmaf(part[s * a.D + lane + 64], w, o1);
  }
  sum[wave][lane] = o0;
  sum[wave][lane + 64] = o1;
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= a.D) return;
  float o = 0.f;
#pragma unroll
  for (int w = 0; w < JW; ++w) o += sum[w][d];
  put<E>(a.o, row / a.H * a.o_sb + row % a.H * a.o_sh + d, lt == 0.f ? 0.f : o / lt);
}

template <typename E, int D>
hipError_t launch_d(const DecodeArgs& a, bool cap, hipStream_t st) {
  const dim3 grid(a.B * a.Hk * ((a.G + 31) / 32), a.splits), block(64 * kWaves<E, D>);
  if (cap && a.slopes)
    hipLaunchKernelGGL((decode_kernel<E, D, true, true>), grid, block, 0, st, a);
  else if (cap)
    hipLaunchKernelGGL((decode_kernel<E, D, true, false>), grid, block, 0, st, a);
  else if (a.slopes)
    hipLaunchKernelGGL((decode_kernel<E, D, false, true>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((decode_kernel<E, D, false, false>), grid, block, 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  static_assert(kMaxParts == 64, "four parts to a wave");
  if (a.splits <= 16)
    hipLaunchKernelGGL((decode_join_kernel<E, 4>), dim3(a.B * a.H), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((decode_join_kernel<E, 16>), dim3(a.B * a.H), dim3(1024), 0, st, a);
  return hipGetLastError();
}

template <typename E>
hipError_t launch_e(const DecodeArgs& a, bool cap, hipStream_t st) {
  return a.D <= 64 ? launch_d<E, 64>(a, cap, st) : launch_d<E, 128>(a, cap, st);
}

}  // namespace

// Parts the keys are split into: four workgroups per CU, so that sequences of
// different lengths even out, at least four tiles of 64 keys to a part.
int decode_splits(int dtype, int B, int H, int Hk, int S, int D) {
  const int64_t wgs = (int64_t)B * Hk * ((H / Hk + 31) / 32);
  const int64_t want = (1024 + wgs - 1) / wgs, most = ((int64_t)S + 255) / 256;
  const int64_t n = want < most ? want : most;
  return n > kMaxParts ? kMaxParts : (int)n;
}

hipError_t launch_decode(int dtype, const DecodeArgs& a, bool cap, hipStream_t st) {
  if (dtype == 0) return launch_e<F32>(a, cap, st);
  return dtype == 1 ? launch_e<F16>(a, cap, st) : launch_e<BF16>(a, cap, st);
}

}  // namespace mi
