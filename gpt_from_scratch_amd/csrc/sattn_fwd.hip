// sattn_fwd.hip — forward of attention with modified scores (capped, biased by
// distance, masked by documents or a prefix, key heads shared by query heads),
// for bf16, f16 and fp32.  The mathematics is at the top of sattn_device.h.
//
// Bound by the matrix cores for plain scores; a cap adds two transcendentals per
// score to the softmax's one, which take longer than the score's products.  Causal
// B2 H16/4 S4096 D128 141-145 us (950-975 TFLOP/s); B1 H32/8 S4096 D128 with a cap
// 168 us; B8 H12 S1024 D64 with slopes 28 us; fp32 B2 H12 S1000 D64, prefix 46 us.
//
// Work decomposition, as in attn_fwd.hip: a workgroup (4 waves) owns 128 query
// rows of one head, wave w rows [32w, 32w + 32); S^T = K Q^T and O^T = V^T P^T
// keep a query per lane, so the softmax's statistics are per-lane scalars and P
// feeds the second product from the accumulators; 64-key tiles of K and V come
// in by direct global -> LDS loads, double buffered, one barrier per tile.
//   * Which key tiles a workgroup visits is listed beforehand
//     (TileWalk) from positions, the prefix and the 64-key ranges of document
//     ids: tiles without a visible pair cost nothing, tiles where every pair is
//     visible run without mask code.
//   * Query heads that share a key head go to the same XCD (workgroups are dealt
//     round robin over the 8 XCDs), so that its L2 reads K and V once for all.
//   * Small grids split a query tile's keys into parts (fwd_parts), joined by a second
//     launch.
//   * Head dims below 64 and between 64 and 128 run in the next layout with zero
//     chunks.
#include <type_traits>

#include "sattn_device.h"

namespace mi {

namespace {

// Document id ranges of each 64 keys and each 64 queries: a wave per record.
__global__ __launch_bounds__(256) void doc_tiles_kernel(const int* docs, DocTile* out, int B, int Sq,
                                                        int Sk, int nk, int nq) {
  const int lane = threadIdx.x & 63;
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= (int64_t)B * (nk + nq)) return;
  const bool key = i < (int64_t)B * nk;
  const int64_t j = key ? i : i - (int64_t)B * nk;
  const int per = key ? nk : nq, b = (int)(j / per), t = (int)(j % per);
  const int off = key ? 0 : Sk - Sq, rows = key ? Sk : Sq;
  const DocRange r = doc_range(docs + (int64_t)b * Sk, off + 64 * t, min(64, rows - 64 * t), lane);
  const int lo[2] = {r.block_lo(0), r.block_lo(1)}, hi[2] = {r.block_hi(0), r.block_hi(1)};
  if (lane == 0) out[i] = DocTile{min(lo[0], lo[1]), max(hi[0], hi[1]), r.pad != 0, 0};
}

// A wave's O (normalised) and lse.  A row without a visible key: O = 0, lse = -inf.
template <typename E, int D>
__device__ __forceinline__ void finish_rows(const SAttnArgs& a, int b, int h, int qw,
                                            const f32x16 (&acc)[D / 32], float m, float l,
                                            char* stage) {
  using L = Lay<E, D>;
  const int lane = threadIdx.x & 63, qrow = qw + (lane & 31), nrows = min(32, a.Sq - qw);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t at = (b * a.o.sb + h * a.o.sh + qw * a.o.ss) * L::ESZ, row = a.o.ss * L::ESZ;
  store_rows<E, D>(acc, inv, stage, (char*)a.o.ptr + at, row, a.dch, nrows);
  if constexpr (L::ESZ == 2)
    if (a.olo) store_rows<E, D, true>(acc, inv, stage, (char*)a.olo + at, row, a.dch, nrows);
  if (lane < 32 && qrow < a.Sq)
    a.lse[((int64_t)b * a.H + h) * a.Sq + qrow] =
        l == 0.f ? -INFINITY : (m + fast_log2(l)) * kLn2;
}

constexpr float kSlack = 8.f;  // log2 units a score may exceed the running reference by

// Waves per SIMD the register budget is held to.  Documents: one fewer, or the mask's ids
// cost spills in every step (B8 H24 S1024 D64, 4 documents: 46 us against 30.5).
template <typename E, int D, bool BIAS, bool DOCS, int KS>
constexpr int kFwdWaves = Lay<E, D>::RB > 256   ? 1
                          : Lay<E, D>::RB > 128 ? 2
                                                : (BIAS ? 3 : 4) - (DOCS && KS == 1 ? 1 : 0);

// DOCS: with document ids.  Without, the code for them is not there at all: 2 to 8% (B8 H12
// S1024 D64 24.3 -> 22.6 us, B2 H16/4 S2048 D128 53.5 -> 51.9).
// KS = 2: a wave takes one 32-key block of each tile instead of both, two waves share
// 32 query rows and merge at the end, and a workgroup owns 64 rows (see key_split).
template <typename E, int D, bool CAP, bool BIAS, bool DOCS, int KS>
__global__ __launch_bounds__(256, (kFwdWaves<E, D, BIAS, DOCS, KS>)) void sattn_fwd_kernel(SAttnArgs a) {
  using L = Lay<E, D>;
  constexpr int BQ = 128 / KS, BK = 64, NB = 2 / KS;
  __shared__ __attribute__((aligned(16))) char K0[BK * L::RB];
  __shared__ __attribute__((aligned(16))) char K1[BK * L::RB];
  __shared__ __attribute__((aligned(16))) char V0[BK * L::RB];
  __shared__ __attribute__((aligned(16))) char V1[BK * L::RB];
  __shared__ __attribute__((aligned(16))) int I0[BK];  // document ids of the keys
  __shared__ __attribute__((aligned(16))) int I1[BK];
  __shared__ int list[kListed];

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Sq = a.Sq, Sk = a.Sk;

  // last query tiles first (the longest under a causal mask); within a tile, key
  // heads run fastest, then the query heads of a group
  const int BH = a.B * a.H, BHk = a.B * a.Hk;
  const int nqt = (Sq + BQ - 1) / BQ;
  const int part = blockIdx.x / BH % a.parts, qt = nqt - 1 - blockIdx.x / BH / a.parts;
  const int n = blockIdx.x % BH, bk = n % BHk, b = bk / a.Hk, hk = bk % a.Hk;
  const int h = hk * a.G + n / BHk;

  const int q0 = qt * BQ, qw = q0 + 32 * (wave / KS), qrow = qw + l32, qpos = a.off + qrow;
  const int slice = KS == 1 ? 0 : wave & 1;
  const bool wave_valid = qw < Sq;
  const int* docs = DOCS ? a.docs + (int64_t)b * Sk : nullptr;
  const int prefix = a.prefix ? max(a.prefix[b], 0) : 0;
  const float slope2 = BIAS ? a.slopes[h] * kLog2e : 0.f;

  const char* qp = (const char*)a.q.ptr + (b * a.q.sb + h * a.q.sh + qrow * a.q.ss) * L::ESZ;
  u32x4 qf[L::KS];
#pragma unroll
  for (int ks = 0; ks < L::KS; ++ks)
    qf[ks] = qrow < Sq && 2 * ks + g < a.dch ? *(const u32x4*)(qp + 16 * (2 * ks + g))
                                              : u32x4{0, 0, 0, 0};
  const int qdoc = DOCS && qrow < Sq ? docs[qpos] : 0;
  // last key that position and sequence end leave visible; none for padding
  int klast = Sk - 1, wlast = Sk - 1;
  if (a.causal) {
    klast = min(max(qpos, prefix - 1), Sk - 1);
    wlast = max(a.off + min(qw + 31, Sq - 1), prefix - 1);
  }
  if (qdoc < 0) klast = -1;

  const int pmin = a.off + q0, pmax = a.off + min(q0 + BQ, Sq) - 1;
  DocRange own = {};
  if (DOCS) own = doc_range(docs, pmin, pmax - pmin + 1, lane);
  const DocTile* ktiles = a.ktiles + (int64_t)b * ((Sk + BK - 1) / BK);
  const int kend = a.causal ? min(max(pmax + 1, prefix), Sk) : Sk, ntiles = (kend + BK - 1) / BK;
  // full: all keys before every query of the workgroup, or in the prefix
  const int kfull = a.causal ? min(max(pmin + 1, prefix), Sk) : Sk;
  auto look = [&](int t) __attribute__((always_inline)) {
    int f = doc_bits(ktiles[t], own);
#pragma unroll
    for (int i = 0; i < 4 / KS; ++i) {
      const int seen = a.causal ? max(pmin + 32 * i + 1, prefix) : Sk;  // of block i's first row
      if ((t + 1) * BK > min(seen, Sk)) f &= ~(kFull << i);
    }
    return f;
  };

  Stage<E, D, BK> ksrc, vsrc;
  ksrc.init(a.k, b, hk, a.dch, lane, wave);
  vsrc.init(a.v, b, hk, a.dch, lane, wave);
  Reads<E, D> rd;
  rd.init(lane, slice);

  auto fetch = [&](int t, char* kb, char* vb, int* ib) __attribute__((always_inline)) {
    const int k0 = (t & kTileIndex) * BK;
    if (DOCS && (t & kPad)) {
      ksrc.load_padded(k0, Sk, kb, lane, wave, docs + k0);
      vsrc.load_padded(k0, Sk, vb, lane, wave, docs + k0);
    } else {
      ksrc.load(k0, Sk, kb, wave);
      vsrc.load(k0, Sk, vb, wave);
    }
    if (DOCS && wave == 0)
      buffer_load_lds4(tile_rsrc(docs + k0, 4 * min(BK, Sk - k0)), 4 * lane, (float*)ib);
  };

  f32x16 acc[L::DB];
#pragma unroll
  for (int i = 0; i < L::DB; ++i) acc[i] = f32x16{};
  float m_run = -INFINITY, l_run = 0.f;
  const float c = BIAS ? 1.f : a.sc.f;  // factor of y below
  // with a causal mask alone no visible key is ahead of its query
  const bool one_sided = BIAS && a.causal && !a.prefix;
  const float gstep = one_sided ? slope2 : 0.f;
  // A wave in its P V products goes before one in its softmax, whose time the products
  // hide: B2 H16/4 S4096 D128 155 -> 141 us, with a bias 173 -> 161.  With a cap the
  // softmax is the longer part and must not wait (172 -> 182).
  constexpr bool kPrio = !CAP;

  auto step = [&](int cur, int nxt, auto slot) __attribute__((always_inline)) {
    constexpr int I = decltype(slot)::value;
    const char* kt = I ? K1 : K0;
    const char* vt = I ? V1 : V0;
    const int* it = I ? I1 : I0;
    if (nxt >= 0) fetch(nxt, I ? K0 : K1, I ? V0 : V1, I ? I0 : I1);
    rd.refresh();
    const int k0 = (cur & kTileIndex) * BK + 32 * slice;  // the wave's first key
    if (wave_valid && (!DOCS || (cur & kLive << wave / KS)) && k0 <= wlast) {
      f32x16 s[NB];
#pragma unroll
      for (int ks = 0; ks < L::KS; ++ks)
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
          s[kb] = Elem<E>::mfma(rd.row(kt, kb, ks), qf[ks], ks == 0 ? f32x16{} : s[kb]);
      // y: scores as f * y + base (+ the group's step, below) in log2 units
      float base = a.sc.b0;
      if constexpr (CAP || BIAS) {
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kb][r] = score_y<E, CAP>(s[kb][r], a.sc);
      }
      if constexpr (BIAS) {
        const float d0 = (float)(qpos - k0 - 4 * g);
        if (one_sided) {
          // key k0 + 4 g + n (n = 8 m + i) is d0 - n behind: -slope2 d0 goes into the
          // base, slope2 i into y, slope2 8 m into the group of four registers
          base -= slope2 * d0;
#pragma unroll
          for (int kb = 0; kb < NB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              s[kb][r] = __builtin_fmaf(s[kb][r], a.sc.f, slope2 * (float)(r & 3));
        } else {
#pragma unroll
          for (int kb = 0; kb < NB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              s[kb][r] = __builtin_fmaf(
                  -slope2, __builtin_fabsf(d0 - (32 * kb + 8 * (r >> 2) + (r & 3))),
                  s[kb][r] * a.sc.f);
        }
      }
      if (!(cur & kFull << wave / KS)) {
        const int rel = klast - k0 - 4 * g;
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (32 * kb + 8 * (r >> 2) + (r & 3) > rel) s[kb][r] = -INFINITY;
        if (DOCS) {
#pragma unroll
          for (int kb = 0; kb < NB; ++kb)
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
              const i32x4 d4 = *(const i32x4*)(it + 32 * (slice + kb) + 8 * jj + 4 * g);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (d4[i] != qdoc) s[kb][4 * jj + i] = -INFINITY;
            }
        }
      }
      float mx;
      if constexpr (BIAS) {
        mx = -INFINITY;
#pragma unroll
        for (int m = 0; m < 4 * NB; ++m) {
          const f32x16& x = s[m >> 2];
          const int r = 4 * (m & 3);
          mx = vmax(mx, vmax(vmax(x[r], x[r + 1]), vmax(x[r + 2], x[r + 3])) + gstep * (8 * m));
        }
      } else {
        mx = vmax(s[0][0], s[0][1]);
#pragma unroll
        for (int i = 2; i < 16 * NB; i += 2)
          mx = vmax(vmax(mx, s[i >> 4][i & 15]), s[i >> 4][(i & 15) + 1]);
      }
      mx = max_halves(__builtin_fmaf(mx, c, base));  // (base is the half's own)
      // The reference moves only when a score passes it by more than kSlack:
      // P stays below 2^8, and O and l share the reference whatever it is.
      if (__any(mx > m_run + kSlack)) {
        const float m_new = fmaxf(m_run, mx);
        const float alpha = fast_exp2(m_run - (m_new == -INFINITY ? 0.f : m_new));
        l_run *= alpha;
#pragma unroll
        for (int db = 0; db < L::DB; ++db) acc[db] *= alpha;
        m_run = m_new;
      }
      // (0 for a row that has seen no key yet)
      const float ref = (m_run == -INFINITY ? 0.f : m_run) - base;
      u32x4 p[NB][L::NG];
      float ps[2] = {0.f, 0.f};
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if constexpr (BIAS)
            s[kb][r] = fast_exp2(s[kb][r] - (ref - gstep * (32 * kb + 8 * (r >> 2))));
          else
            s[kb][r] = fast_exp2(__builtin_fmaf(s[kb][r], c, -ref));
          // the sum before P is rounded for the product: lse is an fp32 result
          ps[r & 1] += s[kb][r];
        }
#pragma unroll
        for (int ng = 0; ng < L::NG; ++ng) p[kb][ng] = Elem<E>::operand(s[kb], ng);
      }
      l_run += ps[0] + ps[1];
      if constexpr (kPrio) __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int ng = 0; ng < L::NG; ++ng)
#pragma unroll
          for (int db = 0; db < L::DB; ++db)
            acc[db] = Elem<E>::mfma(rd.col(vt, kb, ng, db), p[kb][ng], acc[db]);
      if constexpr (kPrio) __builtin_amdgcn_s_setprio(0);
    }
    __syncthreads();
  };
  for (int first = 0; first < ntiles; first += kListed) {
    TileWalk walk;
    if (DOCS) {
      walk.list = list;
      walk.count = tile_list(list, first, ntiles, look);
    } else {
      walk.list = nullptr;
      walk.lo = walk.f0 = first;
      walk.f1 = kfull / BK;
      walk.count = min(ntiles - first, kListed);
    }
    walk.begin(part, a.parts, 0, 1);
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

  float l = sum_halves(l_run);
  char* stage = wave == 0 ? K0 : wave == 1 ? K1 : wave == 2 ? V0 : V1;
  if constexpr (KS > 1) {
    // the second wave of a pair hands over, the first takes both to the common reference
    __shared__ float ml[2][2][64];
    float* const other = (float*)(wave < 2 ? K0 : K1);
    float(&pml)[2][64] = ml[wave >> 1];
    if (slice) {
      part_store<L::DB>(acc, (f32x4*)other, lane);
      pml[0][lane] = m_run;
      pml[1][lane] = l;
    }
    __syncthreads();
    if (slice) return;
    const float m1 = pml[0][lane], m = fmaxf(m_run, m1), ref = m == -INFINITY ? 0.f : m;
    const float f0 = fast_exp2(m_run - ref), f1 = fast_exp2(m1 - ref);
#pragma unroll
    for (int db = 0; db < L::DB; ++db) acc[db] *= f0;
    part_add<L::DB>(acc, (const f32x4*)other, lane, f1);
    l = __builtin_fmaf(l, f0, pml[1][lane] * f1);
    m_run = m;
    stage = wave == 0 ? V0 : V1;
  }
  if (!wave_valid) return;
  if (a.parts > 1) {
    const int64_t at = ((int64_t)(qw / 32) * BH + b * a.H + h) * a.parts + part;
    part_store<L::DB>(acc, part_at<L::DB>(a.part, at), lane);
    float* ml = a.ml + at * 64;
    if (g == 0) {
      ml[l32] = m_run;
      ml[32 + l32] = l;
    }
    return;
  }
  finish_rows<E, D>(a, b, h, qw, acc, m_run, l, stage);
}

// O and lse of query tiles split into parts: each row's parts taken to their common
// reference and added in order.
template <typename E, int D>
__global__ __launch_bounds__(256) void sattn_join_kernel(SAttnArgs a) {
  using L = Lay<E, D>;
  __shared__ __attribute__((aligned(16))) char stage[4][32 * L::RB];
  const int lane = threadIdx.x & 63, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int BH = a.B * a.H, qt = blockIdx.x / BH, bh = blockIdx.x % BH, qw = qt * 128 + 32 * wave;
  if (qw >= a.Sq) return;
  const int64_t at = ((int64_t)(qw / 32) * BH + bh) * a.parts;
  float m = -INFINITY;
  for (int i = 0; i < a.parts; ++i) m = fmaxf(m, a.ml[(at + i) * 64 + l32]);
  const float ref = m == -INFINITY ? 0.f : m;
  f32x16 acc[L::DB];
#pragma unroll
  for (int i = 0; i < L::DB; ++i) acc[i] = f32x16{};
  float l = 0.f;
  for (int i = 0; i < a.parts; ++i) {
    const float* ml = a.ml + (at + i) * 64;
    const float w = fast_exp2(ml[l32] - ref);
    l = __builtin_fmaf(ml[32 + l32], w, l);
    part_add<L::DB>(acc, part_at<L::DB>(a.part, at + i), lane, w);
  }
  finish_rows<E, D>(a, bh / a.H, bh % a.H, qw, acc, m, l, stage[wave]);
}

int64_t tiles128(const SAttnArgs& a) { return (int64_t)((a.Sq + 127) / 128) * a.B * a.H; }

// Whether two waves share a query row's keys: while workgroups are few, shorter steps
// and twice the workgroups (as attn_fwd.hip's key_split).  Documents leave short
// chains of different lengths, and at D <= 64 the split evens them out up to twice as
// many (us whole / split, 768 and 1024 tiles: 29.1 / 24.9, 43.6 / 37.0; at D = 128,
// 1024 tiles: 57 / 70, 82 / 85).
bool key_split(const SAttnArgs& a) {
  if (a.docs && a.D <= 64) return tiles128(a) <= 1024;
  return tiles128(a) <= (!a.causal ? 128 : a.D > 64 ? 256 : 512);
}

// Parts a query tile's keys are split into.  A workgroup is a serial chain of key
// tiles, and a launch of few of them leaves the chip empty; a split costs writing
// and reading the parts' fp32 O once.  Up to one workgroup per CU, two where chains
// are 32 tiles or longer and the join matters less (B1 H4 S4096 D64: 29 us against
// 42), three for fp32, whose products take sixteen times as long; no fewer than four
// key tiles to a part.
int fwd_parts(const SAttnArgs& a, bool f32) {
  const int64_t n = tiles128(a) * (key_split(a) ? 2 : 1);
  const int64_t most = (a.Sk + 255) / 256, want = (f32 ? 768 : a.Sk >= 2048 ? 512 : 256) / n;
  return (int)(want < 2 ? 1 : want < most ? want : most);
}

template <typename E, int D, int KS>
hipError_t launch_k(const SAttnArgs& a, bool cap, hipStream_t st) {
  const dim3 grid((a.Sq + 128 / KS - 1) / (128 / KS) * a.B * a.H * a.parts), block(256);
  const bool docs = a.docs;
  auto run = [&](auto c, auto b) {
    constexpr bool C = decltype(c)::value, B = decltype(b)::value;
    if (docs) hipLaunchKernelGGL((sattn_fwd_kernel<E, D, C, B, true, KS>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((sattn_fwd_kernel<E, D, C, B, false, KS>), grid, block, 0, st, a);
  };
  if (cap && a.slopes) run(std::true_type{}, std::true_type{});
  else if (cap) run(std::true_type{}, std::false_type{});
  else if (a.slopes) run(std::false_type{}, std::true_type{});
  else run(std::false_type{}, std::false_type{});
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.parts == 1) return e;
  hipLaunchKernelGGL((sattn_join_kernel<E, D>), dim3((a.Sq + 127) / 128 * a.B * a.H), block, 0, st,
                     a);
  return hipGetLastError();
}

template <typename E, int D>
hipError_t launch_d(const SAttnArgs& a, bool cap, hipStream_t st) {
  return key_split(a) ? launch_k<E, D, 2>(a, cap, st) : launch_k<E, D, 1>(a, cap, st);
}

template <typename E>
hipError_t launch_e(const SAttnArgs& a, bool cap, hipStream_t st) {
  return a.D <= 64 ? launch_d<E, 64>(a, cap, st) : launch_d<E, 128>(a, cap, st);
}

}  // namespace

hipError_t launch_doc_tiles(const int* docs, void* tiles, int B, int Sq, int Sk, hipStream_t st) {
  const int nk = (Sk + 63) / 64, nq = (Sq + 63) / 64;
  const int64_t n = (int64_t)B * (nk + nq);
  hipLaunchKernelGGL(doc_tiles_kernel, dim3((uint32_t)((n + 3) / 4)), dim3(256), 0, st, docs,
                     (DocTile*)tiles, B, Sq, Sk, nk, nq);
  return hipGetLastError();
}

void sattn_fwd_split(int dtype, SAttnArgs& a, float* ws, int64_t* elems) {
  const int64_t blocks = 4 * tiles128(a);  // of 32 rows
  const int64_t per = 32 * (a.D <= 64 ? 64 : 128);
  a.parts = fwd_parts(a, dtype == 0);
  if (elems) *elems = a.parts > 1 ? blocks * a.parts * (per + 64) : 0;
  a.part = ws;
  a.ml = ws + blocks * a.parts * per;
}

hipError_t launch_sattn_fwd(int dtype, const SAttnArgs& a, bool cap, hipStream_t st) {
  if (dtype == 0) return launch_e<F32>(a, cap, st);
  return dtype == 1 ? launch_e<F16>(a, cap, st) : launch_e<BF16>(a, cap, st);
}

}  // namespace mi
