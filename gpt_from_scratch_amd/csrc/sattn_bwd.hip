// sattn_bwd.hip — backward of attention with modified scores, for bf16, f16 and
// fp32 (sattn_device.h has the forward's mathematics).  With lse from before and
// delta = rowsum(dO * O):
//   P = exp(x - lse);  dV = P^T dO;  dP = dO V^T;  dx = P * (dP - delta)
//   dz = dx * (1 - tanh^2(z / cap));  dQ = scale * dz K;  dK = scale * dz^T Q
// dK and dV of a key head sum over the query heads that share it.
//
// Two kinds of work item in one launch, as in attn_bwd.hip, both without atomics,
// so results repeat bit for bit:
//   dK/dV: 128 keys of one key head, looping over the group's query heads and
//     their query tiles; S = Q K^T and dP = dO V^T keep a key per lane, so P and
//     dz feed dV^T = dO^T P and dK^T = Q^T dz from the accumulators.  The dP
//     accumulators start at +delta and V is negated, so they end at delta - dP;
//   dQ: 128 queries of one head, looping over key tiles; a query per lane.
// S and dP are formed twice, 7 products where 5 would do, in exchange for no
// atomics on dQ.  Tiles without a visible pair are not visited, as in the forward
// (TileWalk).  An item that would be too long a chain for the size of the launch is
// split into parts (parts_of), whose fp32 sums a last launch adds up in order.
//
// Bound by a step's latency (read, product, exponential, product) at two waves per
// SIMD: causal B2 H16/4 S4096 D128 540-580 us (590-640 TFLOP/s counting 5 products),
// B8 H12 S1024 D64 with slopes 81 us, fp32 B2 H12 S1000 D64 with a prefix 144 us.
//
// delta subtracts from dP what O says, so O's rounding would reach every dz of a
// row: the forward keeps what the rounding left (olo), and delta is as exact as fp32
// sums are.
#include <type_traits>

#include "sattn_device.h"

namespace mi {

namespace {

// Rows of a streamed tile: two tiles of two tensors, twice buffered.
template <typename E, int D>
constexpr int kTile = Lay<E, D>::RB > 128 ? 32 : 64;

template <typename E, int D>
constexpr int kWavesPerSimd = Lay<E, D>::RB > 256 ? 1 : 2;

__device__ __forceinline__ const char* head_bytes(const TensorArg& t, int b, int h, int esz) {
  return (const char*)t.ptr + (b * t.sb + h * t.sh) * esz;
}

// A wave's own 32 rows as B operands: lane: row l32, chunk 2 ks + g.
template <typename E, int D>
__device__ __forceinline__ void load_own(const TensorArg& t, int b, int h, int row, bool valid,
                                         int dch, int g, u32x4 (&x)[Lay<E, D>::KS]) {
  using L = Lay<E, D>;
  const char* p = head_bytes(t, b, h, L::ESZ) + row * t.ss * L::ESZ;
#pragma unroll
  for (int ks = 0; ks < L::KS; ++ks)
    x[ks] = valid && 2 * ks + g < dch ? *(const u32x4*)(p + 16 * (2 * ks + g)) : u32x4{0, 0, 0, 0};
}

// Whether the rows' lse2 holds the bias of their place in a block (sattn_delta_kernel).
template <typename E>
__device__ __forceinline__ bool lse_ramp(const SAttnArgs& a) {
  return Elem<E>::kBytes == 2 && a.slopes && a.causal && !a.prefix;
}

// ---------------------------------------------------------------------------
// delta, and lse * log2(e) less the scores' constant
// ---------------------------------------------------------------------------
// Eight lanes per row, R rows per lane with all their loads in flight (us for R = 1, 2, 4:
// B8 H12 S1024 D64 9.1, 8.4, 9.4 for 38 MB; B2 H16 S4096 D128 16.5, 17.2, 17.9 for 101 MB;
// fp32 B2 H12 S1000 D64 4.2, 4.6, 5.0).
// Where no visible key is ahead of its query, and to the 16-bit types, which can
// afford its rounding, the distance bias's part of the row's place in its block of 32
// goes into lse2 here, once per row instead of once per score of dK / dV.
template <typename E, int D, int R>
__global__ __launch_bounds__(256) void sattn_delta_kernel(SAttnArgs a, uint32_t rows, FastDiv dS,
                                                          FastDiv dH) {
  constexpr int ESZ = Elem<E>::kBytes, NC = D * ESZ / 16 / 8;
  const int sub = threadIdx.x % 8;
  u32x4 x[R][NC], y[R][NC], z[R][NC];
  float ramp[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const uint32_t row = blockIdx.x * (32u * R) + 32 * i + threadIdx.x / 8;
    const uint32_t bh = fdiv(row, dS), s = row - bh * dS.d, b = fdiv(bh, dH), h = bh - b * dH.d;
    const int64_t at = (b * a.o.sb + h * a.o.sh + s * a.o.ss) * ESZ;
    const u32x4* o = (const u32x4*)((const char*)a.o.ptr + at);
    const u32x4* lo = a.olo ? (const u32x4*)((const char*)a.olo + at) : nullptr;
    const u32x4* d = (const u32x4*)((const char*)a.dout.ptr +
                                    (b * a.dout.sb + h * a.dout.sh + s * a.dout.ss) * ESZ);
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int c = sub + 8 * n;
      const bool have = row < rows && c < a.dch;
      x[i][n] = have ? o[c] : u32x4{0, 0, 0, 0};
      y[i][n] = have ? d[c] : u32x4{0, 0, 0, 0};
      z[i][n] = have && lo ? lo[c] : u32x4{0, 0, 0, 0};
    }
    ramp[i] = lse_ramp<E>(a) && row < rows ? a.slopes[h] * kLog2e * (float)(s & 31) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const uint32_t row = blockIdx.x * (32u * R) + 32 * i + threadIdx.x / 8;
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t u = x[i][n][k], v = y[i][n][k], w = z[i][n][k];
        if constexpr (ESZ == 4) {
          sum = __builtin_fmaf(__uint_as_float(u), __uint_as_float(v), sum);
        } else {
          sum = __builtin_fmaf(E::to_f32(u & 0xffff) + E::to_f32(w & 0xffff), E::to_f32(v & 0xffff),
                               sum);
          sum = __builtin_fmaf(E::to_f32(u >> 16) + E::to_f32(w >> 16), E::to_f32(v >> 16), sum);
        }
      }
    sum = group_sum<8>(sum);
    if (row < rows && sub == 0) {
      const_cast<float*>(a.delta)[row] = sum;
      const_cast<float*>(a.lse2)[row] = a.lse[row] * kLog2e - a.sc.b0 + ramp[i];
    }
  }
}

// ---------------------------------------------------------------------------
// dK, dV
// ---------------------------------------------------------------------------
// Two tiles of each streamed tensor, per-row values of the queries, own rows of K.
struct Buffers {
  char *A0, *A1, *B0, *B1;
  float *S0, *S1;  // lse2, delta, document ids; for dQ: document ids
  char* own;
  int* list;       // see TileWalk
};

template <typename E, int D, bool CAP, bool BIAS, bool DOCS>
__device__ __forceinline__ void dkdv_item(const SAttnArgs& a, int item, const Buffers& buf) {
  using L = Lay<E, D>;
  constexpr int OWN = 128, T = kTile<E, D>, TB = T / 32;
  constexpr bool K_IN_LDS = L::RB > 128;  // K and V rows and both sums pass 256 registers
  char *const Q0 = buf.A0, *const Q1 = buf.A1, *const G0 = buf.B0, *const G1 = buf.B1;
  float *const S0 = buf.S0, *const S1 = buf.S1;

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Sq = a.Sq, Sk = a.Sk;
  const int BHk = a.B * a.Hk;
  // key tile 0 sees the most queries under a causal mask: first
  const int kt = item / BHk / a.parts, part = item / BHk % a.parts, bk = item % BHk,
            b = bk / a.Hk, hk = bk % a.Hk;
  const int k0 = kt * OWN, kw = k0 + 32 * wave, krow = kw + l32;
  const bool wave_valid = kw < Sk;
  const int* docs = DOCS ? a.docs + (int64_t)b * Sk : nullptr;
  const int prefix = a.prefix ? max(a.prefix[b], 0) : 0;
  const int kdoc = DOCS && krow < Sk ? docs[krow] : 0;
  // first query position that sees this lane's key, and the wave's first
  int qfirst = 0, wfirst = 0;
  if (a.causal) {
    qfirst = krow < prefix ? 0 : krow;
    wfirst = kw < prefix ? 0 : kw;
  }
  if (kdoc < 0) qfirst = 0x7fffffff;

  char* const kl = buf.own + (K_IN_LDS ? wave * 32 * L::RB : 0);
  u32x4 kf[L::KS], vn[L::KS];
  load_own<E, D>(a.k, b, hk, krow, krow < Sk, a.dch, g, kf);
  load_own<E, D>(a.v, b, hk, krow, krow < Sk, a.dch, g, vn);
  constexpr uint32_t neg = L::ESZ == 2 ? 0x80008000u : 0x80000000u;
#pragma unroll
  for (int ks = 0; ks < L::KS; ++ks) vn[ks] ^= neg;
  Reads<E, D> rd;
  rd.init(lane);
  if constexpr (K_IN_LDS) {
#pragma unroll
    for (int ks = 0; ks < L::KS; ++ks)
      *(u32x4*)(kl + 256 * (ks / rd.NR) + rd.r[ks % rd.NR]) = kf[ks];
  }

  const int kmax = min(k0 + OWN, Sk) - 1;
  DocRange own = {};
  if (DOCS) own = doc_range(docs, k0, kmax - k0 + 1, lane);
  const DocTile* qtiles = a.qtiles + (int64_t)b * ((Sq + 63) / 64);
  const int nqt = (Sq + T - 1) / T;
  // first query that sees a key of the workgroup, and the first that sees all of them
  const int qlive = a.causal && k0 >= prefix ? max(k0 - a.off, 0) : 0;
  const int qfull = a.causal && kmax >= prefix ? max(kmax - a.off, 0) : 0;
  auto look = [&](int t) __attribute__((always_inline)) {
    if ((t + 1) * T <= qlive) return 0;
    int f = doc_bits(qtiles[t * T >> 6], own);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int last = min(k0 + 32 * i + 31, Sk - 1);  // of block i
      const int seen = a.causal && last >= prefix ? last - a.off : 0;  // from this query on
      if (t * T < seen || (t + 1) * T > Sq) f &= ~(kFull << i);
    }
    return f;
  };
  Stage<E, D, T> qsrc, gsrc;
  qsrc.init(a.q, b, 0, a.dch, lane, wave);
  gsrc.init(a.dout, b, 0, a.dch, lane, wave);
  const char *qbase = qsrc.base, *gbase = gsrc.base;
  auto fetch = [&](int t, int head, char* qb, char* gb, float* sb) __attribute__((always_inline)) {
    const int q0 = (t & kTileIndex) * T;
    qsrc.base = qbase + head * a.q.sh * L::ESZ;
    gsrc.base = gbase + head * a.dout.sh * L::ESZ;
    if (DOCS && (t & kPad)) {
      qsrc.load_padded(q0, Sq, qb, lane, wave, docs + a.off + q0);
      gsrc.load_padded(q0, Sq, gb, lane, wave, docs + a.off + q0);
    } else {
      qsrc.load(q0, Sq, qb, wave);
      gsrc.load(q0, Sq, gb, wave);
    }
    const int nr = 4 * min(T, Sq - q0);
    const int64_t row = ((int64_t)b * a.H + head) * Sq + q0;
    if (lane < T) {
      if (wave == 0) buffer_load_lds4(tile_rsrc(a.lse2 + row, nr), 4 * lane, sb);
      if (wave == 1) buffer_load_lds4(tile_rsrc(a.delta + row, nr), 4 * lane, sb + T);
      if (wave == 2 && DOCS)
        buffer_load_lds4(tile_rsrc(docs + a.off + q0, nr), 4 * lane, sb + 2 * T);
    }
  };

  f32x16 dk[L::DB], dv[L::DB];
#pragma unroll
  for (int i = 0; i < L::DB; ++i) dk[i] = dv[i] = f32x16{};

  float slope2 = 0.f;
  // with a causal mask alone no visible key is ahead of its query
  const bool one_sided = BIAS && a.causal && !a.prefix;
  auto step = [&](int cur, int nxt, int hnext, auto slot) __attribute__((always_inline)) {
    constexpr int I = decltype(slot)::value;
    const char* qt = I ? Q1 : Q0;
    const char* gt = I ? G1 : G0;
    const float* st = I ? S1 : S0;
    if (nxt >= 0) fetch(nxt, hnext, I ? Q0 : Q1, I ? G0 : G1, I ? S0 : S1);
    rd.refresh();
    const int q0 = (cur & kTileIndex) * T, p0 = a.off + q0;
    if (wave_valid && (!DOCS || (cur & kLive << wave)) && p0 + T - 1 >= wfirst) {
      const bool full = cur & kFull << wave;
      u32x4 pb[TB][L::NG], sb[TB][L::NG];
      f32x16 ss[TB], dps[TB];
#pragma unroll
      for (int qb = 0; qb < TB; ++qb) {
        f32x16 &s = ss[qb], &dp = dps[qb];
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          const f32x4 d4 = *(const f32x4*)(st + T + 32 * qb + 8 * jj + 4 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) dp[4 * jj + i] = d4[i];
        }
#pragma unroll
        for (int ks = 0; ks < L::KS; ++ks)
          s = Elem<E>::mfma(rd.row(qt, qb, ks), K_IN_LDS ? rd.row(kl, 0, ks) : kf[ks],
                            ks == 0 ? f32x16{} : s);
#pragma unroll
        for (int ks = 0; ks < L::KS; ++ks)
          dp = Elem<E>::mfma(rd.row(gt, qb, ks), vn[ks], dp);
      }
#pragma unroll
      for (int qb = 0; qb < TB; ++qb) {
        f32x16 &s = ss[qb], &dp = dps[qb];
        // query of register r: q0 + 32 qb + 8 (r / 4) + 4 g + r % 4, d0 + 8 (r / 4) + r % 4
        // ahead of the lane's key
        const float d0 = (float)(p0 - krow + 32 * qb + 4 * g);
        const float base = -slope2 * (L::ESZ == 2 ? (float)(p0 - krow + 32 * qb) : d0);
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          const f32x4 l4 = *(const f32x4*)(st + 32 * qb + 8 * jj + 4 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 4 * jj + i;
            const float y = score_y<E, CAP>(s[r], a.sc);
            float x;
            if constexpr (BIAS) {
              if (one_sided && L::ESZ == 2)  // the rest is in lse2
                x = __builtin_fmaf(y, a.sc.f, base - l4[i]);
              else if (one_sided)
                x = __builtin_fmaf(y, a.sc.f, base - __builtin_fmaf(slope2, 8 * jj + i, l4[i]));
              else
                x = __builtin_fmaf(y, a.sc.f, __builtin_fmaf(
                        -slope2, __builtin_fabsf(d0 + (8 * jj + i)), -l4[i]));
            } else {
              x = __builtin_fmaf(y, a.sc.f, -l4[i]);
            }
            const float p = fast_exp2(x);
            s[r] = p;
            dp[r] = -(p * dp[r]);
            if constexpr (CAP) dp[r] *= score_slope<E, CAP>(y);
          }
        }
        if (!full) {
          const int base = q0 + 32 * qb + 4 * g;
          // visible: lo <= n < hi, as one unsigned comparison
          const int lo = qfirst == 0x7fffffff ? 64 : max(qfirst - a.off - base, 0);
          const uint32_t span = max(Sq - base - lo, 0);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int n = 8 * (r >> 2) + (r & 3);
            if ((uint32_t)(n - lo) >= span) s[r] = dp[r] = 0.f;
          }
          if (DOCS) {
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
              const i32x4 d4 = *(const i32x4*)(st + 2 * T + 32 * qb + 8 * jj + 4 * g);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (d4[i] != kdoc) s[4 * jj + i] = dp[4 * jj + i] = 0.f;
            }
          }
        }
#pragma unroll
        for (int ng = 0; ng < L::NG; ++ng) {
          pb[qb][ng] = Elem<E>::operand(s, ng);
          sb[qb][ng] = Elem<E>::operand(dp, ng);
        }
      }
#pragma unroll
      for (int qb = 0; qb < TB; ++qb)
#pragma unroll
        for (int ng = 0; ng < L::NG; ++ng)
#pragma unroll
          for (int db = 0; db < L::DB; ++db) {
            dv[db] = Elem<E>::mfma(rd.col(gt, qb, ng, db), pb[qb][ng], dv[db]);
            dk[db] = Elem<E>::mfma(rd.col(qt, qb, ng, db), sb[qb][ng], dk[db]);
          }
    }
    __syncthreads();
  };
  // the group's query heads one after another
  for (int first = 0; first < nqt; first += kListed) {
    TileWalk walk;
    if (DOCS) {
      walk.list = buf.list;
      walk.count = tile_list(buf.list, first, nqt, look);
    } else {
      walk.list = nullptr;
      walk.lo = max(first, qlive / T);
      walk.f0 = (qfull + T - 1) / T;
      walk.f1 = Sq / T;
      walk.count = min(nqt, first + kListed) - walk.lo;
    }
    walk.begin(part, a.parts, hk * a.G, a.G);
    int cur = walk.entry();
    if (cur >= 0) fetch(cur, walk.head, Q0, G0, S0);
    __syncthreads();
    while (cur >= 0) {
      if (BIAS) slope2 = a.slopes[walk.head] * kLog2e;
      walk.step(walk.parts);
      int nxt = walk.entry();
      step(cur, nxt, walk.head, std::integral_constant<int, 0>{});
      if ((cur = nxt) < 0) break;
      if (BIAS) slope2 = a.slopes[walk.head] * kLog2e;
      walk.step(walk.parts);
      nxt = walk.entry();
      step(cur, nxt, walk.head, std::integral_constant<int, 1>{});
      cur = nxt;
    }
  }

  if (!wave_valid) return;
  if (a.parts > 1) {
    const int64_t at = 2 * (((int64_t)(kw / 32) * BHk + bk) * a.parts + part);
    part_store<L::DB>(dv, part_at<L::DB>(a.part, at), lane);
    part_store<L::DB>(dk, part_at<L::DB>(a.part, at + 1), lane);
    return;
  }
  // idle now: the wave's K rows, or one of the tile buffers
  char* stage = K_IN_LDS ? kl : wave == 0 ? Q0 : wave == 1 ? Q1 : wave == 2 ? G0 : G1;
  const int nrows = min(32, Sk - kw);
  store_rows<E, D>(dv, 1.f, stage,
                   (char*)a.dv.ptr + (b * a.dv.sb + hk * a.dv.sh + kw * a.dv.ss) * L::ESZ,
                   a.dv.ss * L::ESZ, a.dch, nrows);
  store_rows<E, D>(dk, a.scale, stage,
                   (char*)a.dk.ptr + (b * a.dk.sb + hk * a.dk.sh + kw * a.dk.ss) * L::ESZ,
                   a.dk.ss * L::ESZ, a.dch, nrows);
}

// ---------------------------------------------------------------------------
// dQ
// ---------------------------------------------------------------------------
template <typename E, int D, bool CAP, bool BIAS, bool DOCS>
__device__ __forceinline__ void dq_item(const SAttnArgs& a, int item, const Buffers& buf) {
  using L = Lay<E, D>;
  constexpr int OWN = 128, T = kTile<E, D>, TB = T / 32;
  char *const K0 = buf.A0, *const K1 = buf.A1, *const V0 = buf.B0, *const V1 = buf.B1;
  int *const I0 = (int*)buf.S0, *const I1 = (int*)buf.S1;

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Sq = a.Sq, Sk = a.Sk;
  const int BH = a.B * a.H, BHk = a.B * a.Hk;
  const int nqt = (Sq + OWN - 1) / OWN;
  const int qt = nqt - 1 - item / BH / a.qparts, part = item / BH % a.qparts;
  const int n = item % BH, bk = n % BHk, b = bk / a.Hk, hk = bk % a.Hk;
  const int h = hk * a.G + n / BHk;
  const int q0 = qt * OWN, qw = q0 + 32 * wave, qrow = qw + l32, qpos = a.off + qrow;
  const bool wave_valid = qw < Sq;
  const int* docs = DOCS ? a.docs + (int64_t)b * Sk : nullptr;
  const int prefix = a.prefix ? max(a.prefix[b], 0) : 0;
  const float slope2 = BIAS ? a.slopes[h] * kLog2e : 0.f;
  const int qdoc = DOCS && qrow < Sq ? docs[qpos] : 0;
  int klast = Sk - 1, wlast = Sk - 1;
  if (a.causal) {
    klast = min(max(qpos, prefix - 1), Sk - 1);
    wlast = max(a.off + min(qw + 31, Sq - 1), prefix - 1);
  }
  if (qdoc < 0) klast = -1;

  u32x4 qf[L::KS], df[L::KS];
  load_own<E, D>(a.q, b, h, qrow, qrow < Sq, a.dch, g, qf);
  load_own<E, D>(a.dout, b, h, qrow, qrow < Sq, a.dch, g, df);
  const int64_t row = ((int64_t)b * a.H + h) * Sq + qrow;
  float lse2 = qrow < Sq ? a.lse2[row] : 0.f;
  if (BIAS && lse_ramp<E>(a)) lse2 -= slope2 * (float)l32;
  const float ndelta = qrow < Sq ? -a.delta[row] : 0.f;

  const int pmin = a.off + q0, pmax = a.off + min(q0 + OWN, Sq) - 1;
  DocRange own = {};
  if (DOCS) own = doc_range(docs, pmin, pmax - pmin + 1, lane);
  const DocTile* ktiles = a.ktiles + (int64_t)b * ((Sk + 63) / 64);
  const int kend = a.causal ? min(max(pmax + 1, prefix), Sk) : Sk, ntiles = (kend + T - 1) / T;
  const int kfull = a.causal ? min(max(pmin + 1, prefix), Sk) : Sk;
  auto look = [&](int t) __attribute__((always_inline)) {
    int f = doc_bits(ktiles[t * T >> 6], own);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int seen = a.causal ? max(pmin + 32 * i + 1, prefix) : Sk;  // of block i's first row
      if ((t + 1) * T > min(seen, Sk)) f &= ~(kFull << i);
    }
    return f;
  };

  Stage<E, D, T> ksrc, vsrc;
  ksrc.init(a.k, b, hk, a.dch, lane, wave);
  vsrc.init(a.v, b, hk, a.dch, lane, wave);
  Reads<E, D> rd;
  rd.init(lane);
  auto fetch = [&](int t, char* kb, char* vb, int* ib) __attribute__((always_inline)) {
    const int k0 = (t & kTileIndex) * T;
    if (DOCS && (t & kPad)) {
      ksrc.load_padded(k0, Sk, kb, lane, wave, docs + k0);
      vsrc.load_padded(k0, Sk, vb, lane, wave, docs + k0);
    } else {
      ksrc.load(k0, Sk, kb, wave);
      vsrc.load(k0, Sk, vb, wave);
    }
    if (DOCS && wave == 0 && lane < T)
      buffer_load_lds4(tile_rsrc(docs + k0, 4 * min(T, Sk - k0)), 4 * lane, (float*)ib);
  };

  f32x16 acc[L::DB];
#pragma unroll
  for (int i = 0; i < L::DB; ++i) acc[i] = f32x16{};
  const bool one_sided = BIAS && a.causal && !a.prefix;
  auto step = [&](int cur, int nxt, auto slot) __attribute__((always_inline)) {
    constexpr int I = decltype(slot)::value;
    const char* kt = I ? K1 : K0;
    const char* vt = I ? V1 : V0;
    const int* it = I ? I1 : I0;
    if (nxt >= 0) fetch(nxt, I ? K0 : K1, I ? V0 : V1, I ? I0 : I1);
    rd.refresh();
    const int k0 = (cur & kTileIndex) * T;
    if (wave_valid && (!DOCS || (cur & kLive << wave)) && k0 <= wlast) {
      u32x4 sb[TB][L::NG];
      f32x16 ss[TB], dps[TB];
#pragma unroll
      for (int kb = 0; kb < TB; ++kb) {
        f32x16 &s = ss[kb], &dp = dps[kb];
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] = ndelta;
#pragma unroll
        for (int ks = 0; ks < L::KS; ++ks)
          s = Elem<E>::mfma(rd.row(kt, kb, ks), qf[ks], ks == 0 ? f32x16{} : s);
#pragma unroll
        for (int ks = 0; ks < L::KS; ++ks) dp = Elem<E>::mfma(rd.row(vt, kb, ks), df[ks], dp);
      }
#pragma unroll
      for (int kb = 0; kb < TB; ++kb) {
        f32x16 &s = ss[kb], &dp = dps[kb];
        const float d0 = (float)(qpos - k0 - 32 * kb - 4 * g);
        const float base = -__builtin_fmaf(slope2, d0, lse2);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float y = score_y<E, CAP>(s[r], a.sc);
          float x;
          if constexpr (BIAS) {
            // the key is d0 - n behind its query, n = 8 (r / 4) + r % 4
            if (one_sided)
              x = __builtin_fmaf(y, a.sc.f, slope2 * (float)(r & 3)) + (base + slope2 * (8 * (r >> 2)));
            else
              x = __builtin_fmaf(y, a.sc.f, __builtin_fmaf(
                      -slope2, __builtin_fabsf(d0 - (8 * (r >> 2) + (r & 3))), -lse2));
          } else {
            x = __builtin_fmaf(y, a.sc.f, -lse2);
          }
          dp[r] *= fast_exp2(x);
          if constexpr (CAP) dp[r] *= score_slope<E, CAP>(y);
        }
        if (!(cur & kFull << wave)) {
          const int rel = klast - k0 - 32 * kb - 4 * g;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (8 * (r >> 2) + (r & 3) > rel) dp[r] = 0.f;
          if (DOCS) {
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
              const i32x4 d4 = *(const i32x4*)(it + 32 * kb + 8 * jj + 4 * g);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (d4[i] != qdoc) dp[4 * jj + i] = 0.f;
            }
          }
        }
#pragma unroll
        for (int ng = 0; ng < L::NG; ++ng) sb[kb][ng] = Elem<E>::operand(dp, ng);
      }
#pragma unroll
      for (int kb = 0; kb < TB; ++kb)
#pragma unroll
        for (int ng = 0; ng < L::NG; ++ng)
#pragma unroll
          for (int db = 0; db < L::DB; ++db)
            acc[db] = Elem<E>::mfma(rd.col(kt, kb, ng, db), sb[kb][ng], acc[db]);
    }
    __syncthreads();
  };
  for (int first = 0; first < ntiles; first += kListed) {
    TileWalk walk;
    if (DOCS) {
      walk.list = buf.list;
      walk.count = tile_list(buf.list, first, ntiles, look);
    } else {
      walk.list = nullptr;
      walk.lo = walk.f0 = first;
      walk.f1 = kfull / T;
      walk.count = min(ntiles - first, kListed);
    }
    walk.begin(part, a.qparts, 0, 1);
    int cur = walk.entry();
    if (cur >= 0) fetch(cur, K0, V0, I0);
    __syncthreads();
    while (cur >= 0) {
      walk.step(walk.parts);
      int nxt = walk.entry();
      step(cur, nxt, std::integral_constant<int, 0>{});
      if ((cur = nxt) < 0) break;
      walk.step(walk.parts);
      nxt = walk.entry();
      step(cur, nxt, std::integral_constant<int, 1>{});
      cur = nxt;
    }
  }

  if (!wave_valid) return;
  if (a.qparts > 1) {
    const int64_t at = ((int64_t)(qw / 32) * BH + b * a.H + h) * a.qparts + part;
    part_store<L::DB>(acc, part_at<L::DB>(a.qpart, at), lane);
    return;
  }
  char* stage = wave == 0 ? K0 : wave == 1 ? K1 : wave == 2 ? V0 : V1;
  store_rows<E, D>(acc, a.scale, stage,
                   (char*)a.dq.ptr + (b * a.dq.sb + h * a.dq.sh + qw * a.dq.ss) * L::ESZ,
                   a.dq.ss * L::ESZ, a.dch, min(32, Sq - qw));
}

// Both kinds in one launch, so that the short items of one fill the gaps that the
// long ones of the other leave.  Runs of 64 workgroups (whole rounds over the XCDs)
// belong to one kind, spread evenly; each kind's own order is longest first.
// DOCS as in the forward (B8 H12 S1024 D64 70 -> 67 us, with slopes 93 -> 86; B2 H16/4
// S4096 D128 with a cap 665 -> 632).
template <typename E, int D, bool CAP, bool BIAS, bool DOCS>
__global__ __launch_bounds__(256, (kWavesPerSimd<E, D>)) void sattn_bwd_kernel(SAttnArgs a, int n0,
                                                                               int n1) {
  using L = Lay<E, D>;
  constexpr int T = kTile<E, D>;
  __shared__ __attribute__((aligned(16))) char A0[T * L::RB];
  __shared__ __attribute__((aligned(16))) char A1[T * L::RB];
  __shared__ __attribute__((aligned(16))) char B0[T * L::RB];
  __shared__ __attribute__((aligned(16))) char B1[T * L::RB];
  __shared__ __attribute__((aligned(16))) float S0[3 * T];
  __shared__ __attribute__((aligned(16))) float S1[3 * T];
  __shared__ __attribute__((aligned(16))) char own[L::RB > 128 ? 128 * L::RB : 16];
  __shared__ int list[kListed];
  const Buffers buf = {A0, A1, B0, B1, S0, S1, own, list};
  const int64_t r0 = (n0 + 63) / 64, r = r0 + (n1 + 63) / 64, t = blockIdx.x / 64;
  const int before = (int)(t * r0 / r);
  const bool dkdv = (t + 1) * r0 / r > before;
  const int item = (dkdv ? before : (int)t - before) * 64 + blockIdx.x % 64;
  if (item >= (dkdv ? n0 : n1)) return;
  if (dkdv)
    dkdv_item<E, D, CAP, BIAS, DOCS>(a, item, buf);
  else
    dq_item<E, D, CAP, BIAS, DOCS>(a, item, buf);
}

// The sums of split items.  Workgroups [0, n0): dV and dK of the key tiles, two
// each; then dQ of the query tiles.
template <typename E, int D>
__global__ __launch_bounds__(256) void sattn_sum_kernel(SAttnArgs a, int n0) {
  using L = Lay<E, D>;
  __shared__ __attribute__((aligned(16))) char stage[4][32 * L::RB];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool query = (int)blockIdx.x >= n0;
  const int which = query ? blockIdx.x - n0 : blockIdx.x >> 1, second = query ? 0 : blockIdx.x & 1;
  const int heads = query ? a.H : a.Hk, n = a.B * heads, tile = which / n, bh = which % n;
  const int rows = query ? a.Sq : a.Sk, row = 128 * tile + 32 * wave;
  if (row >= rows) return;
  f32x16 acc[L::DB];
#pragma unroll
  for (int i = 0; i < L::DB; ++i) acc[i] = f32x16{};
  const int64_t at = (int64_t)(row / 32) * n + bh;
  if (query) {
    for (int i = 0; i < a.qparts; ++i)
      part_add<L::DB>(acc, part_at<L::DB>(a.qpart, at * a.qparts + i), lane, 1.f);
  } else {
    for (int i = 0; i < a.parts; ++i)
      part_add<L::DB>(acc, part_at<L::DB>(a.part, 2 * (at * a.parts + i) + second), lane, 1.f);
  }
  const TensorArg& t = query ? a.dq : second ? a.dk : a.dv;
  store_rows<E, D>(acc, query || second ? a.scale : 1.f, stage[wave],
                   (char*)t.ptr + (bh / heads * t.sb + bh % heads * t.sh + row * t.ss) * L::ESZ,
                   t.ss * L::ESZ, a.dch, min(32, rows - row));
}

template <typename E, int D, bool CAP, bool BIAS, bool DOCS>
hipError_t launch_cb(const SAttnArgs& a, hipStream_t st) {
  const int kitems = (a.Sk + 127) / 128 * a.B * a.Hk, qitems = (a.Sq + 127) / 128 * a.B * a.H;
  const int n0 = kitems * a.parts, n1 = qitems * a.qparts;
  hipLaunchKernelGGL((sattn_bwd_kernel<E, D, CAP, BIAS, DOCS>), dim3(((n0 + 63) / 64 + (n1 + 63) / 64) * 64),
                     dim3(256), 0, st, a, n0, n1);
  const hipError_t e = hipGetLastError();
  const int s0 = a.parts > 1 ? 2 * kitems : 0, s1 = a.qparts > 1 ? qitems : 0;
  if (e != hipSuccess || s0 + s1 == 0) return e;
  hipLaunchKernelGGL((sattn_sum_kernel<E, D>), dim3(s0 + s1), dim3(256), 0, st, a, s0);
  return hipGetLastError();
}

template <typename E, int D>
hipError_t launch_delta(const SAttnArgs& a, hipStream_t st) {
  constexpr int R = D * Elem<E>::kBytes == 128 ? 2 : 1;
  const uint32_t rows = (uint32_t)a.B * a.H * a.Sq;
  hipLaunchKernelGGL((sattn_delta_kernel<E, D, R>), dim3((rows + 32 * R - 1) / (32 * R)), dim3(256), 0,
                     st, a, rows, make_fastdiv(a.Sq), make_fastdiv(a.H));
  return hipGetLastError();
}

template <typename E, int D>
hipError_t launch_d(const SAttnArgs& a, bool cap, hipStream_t st) {
  auto run = [&](auto c, auto b) {
    constexpr bool C = decltype(c)::value, B = decltype(b)::value;
    return a.docs ? launch_cb<E, D, C, B, true>(a, st) : launch_cb<E, D, C, B, false>(a, st);
  };
  if (cap && a.slopes) return run(std::true_type{}, std::true_type{});
  if (cap) return run(std::true_type{}, std::false_type{});
  if (a.slopes) return run(std::false_type{}, std::true_type{});
  return run(std::false_type{}, std::false_type{});
}

template <typename E>
hipError_t launch_e(const SAttnArgs& a, bool cap, hipStream_t st) {
  const hipError_t e = a.D <= 64 ? launch_delta<E, 64>(a, st) : launch_delta<E, 128>(a, st);
  if (e != hipSuccess) return e;
  return a.D <= 64 ? launch_d<E, 64>(a, cap, st) : launch_d<E, 128>(a, cap, st);
}

// Parts of items of `steps` streamed tiles each, when there are n of them: a chain as
// long as the launch has room for, at least four tiles to a part.
// Twice as many with documents, whose items differ more (9 documents of up to 1650 tokens,
// B2 H16/4 S4096 D128: 273 us with 512, 256 with 1024).
int parts_of(int64_t n, int64_t steps, bool docs) {
  const int64_t most = (steps + 3) / 4, want = (docs ? 1024 : 512) / n;
  return (int)(want < 2 ? 1 : want < most ? want : most);
}

}  // namespace

void sattn_bwd_split(SAttnArgs& a, float* ws, int64_t* elems) {
  const int64_t kitems = (int64_t)((a.Sk + 127) / 128) * a.B * a.Hk;
  const int64_t qitems = (int64_t)((a.Sq + 127) / 128) * a.B * a.H;
  const int64_t per = 128 * (a.D <= 64 ? 64 : 128);
  a.parts = parts_of(kitems, (int64_t)(a.Sq + 63) / 64 * a.G, a.docs);
  a.qparts = parts_of(qitems, (a.Sk + 63) / 64, a.docs);
  // delta and lse2, then the parts, 16-byte aligned
  const int64_t rows = ((int64_t)a.B * a.H * a.Sq + 3) / 4 * 4;
  const int64_t p0 = a.parts > 1 ? 2 * kitems * a.parts * per : 0;
  const int64_t p1 = a.qparts > 1 ? qitems * a.qparts * per : 0;
  if (elems) *elems = 2 * rows + p0 + p1;
  a.delta = ws;
  a.lse2 = ws + rows;
  a.part = ws + 2 * rows;
  a.qpart = a.part + p0;
}

hipError_t launch_sattn_bwd(int dtype, const SAttnArgs& a, bool cap, hipStream_t st) {
  if (dtype == 0) return launch_e<F32>(a, cap, st);
  return dtype == 1 ? launch_e<F16>(a, cap, st) : launch_e<BF16>(a, cap, st);
}

}  // namespace mi
