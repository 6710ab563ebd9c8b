// sattn_device.h — pieces shared by the kernels of attention with modified
// scores (sattn_fwd.hip, sattn_bwd.hip, decode.hip).
//
//   z_ij = scale * q_i . k_j            capped: z <- cap * tanh(z / cap)
//   x_ij = z_ij - slope_h * |i - j|     (positions; the last query is the last key)
//   j visible to i iff  document(i) == document(j) >= 0   (where documents are given)
//                  and  (not causal, or j <= i, or j < prefix)
//   P = softmax over the visible j,  O = P V
//
// One code for bf16, f16 and fp32: a tile row is D elements in 16-byte chunks,
// a matrix-core step takes one chunk of each half wave (one 32x32x16 product of
// 16-bit types, four 32x32x2 products of fp32), and the k order inside a step
// is free as long as both operands use the same (see mi_device.h).
#pragma once

#include "mi_device.h"
#include "mi_kernels.h"

namespace mi {

typedef __attribute__((ext_vector_type(4))) int i32x4;

struct F32 {};

template <typename E>
struct Elem {  // 16-bit types
  static constexpr int kBytes = 2;
  static constexpr int kGroups = 2;  // k-groups of a 32-row block, one operand each
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return E::mfma(a, b, c);
  }
  // Operand of k-group n from a 32x32 accumulator (rows 16n .. 16n + 15).  The one
  // rounding of P (and of dS in the backward): the matrix cores take 16-bit operands
  // at sixteen times the fp32 rate.  P is summed before it where lse is a result,
  // after it in decoding, where the sum only divides O.
  static __device__ __forceinline__ u32x4 operand(const f32x16& s, int n) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = E::pack2(s[8 * n + 2 * i], s[8 * n + 2 * i + 1]);
    return w;
  }
  // The operand's values as rounded, summed.
  static __device__ __forceinline__ float sum(u32x4 w, float acc) {
    return E::sum2(w[0], E::sum2(w[1], acc)) + E::sum2(w[2], E::sum2(w[3], 0.f));
  }
  static __device__ __forceinline__ u32x2 pack4(float a, float b, float c, float d) {
    return u32x2{E::pack2(a, b), E::pack2(c, d)};
  }
};

template <>
struct Elem<F32> {
  static constexpr int kBytes = 4;
  static constexpr int kGroups = 4;
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0,
                                               0, 0);
    return c;
  }
  // rows 8n .. 8n + 7
  static __device__ __forceinline__ u32x4 operand(const f32x16& s, int n) {
    return u32x4{__float_as_uint(s[4 * n]), __float_as_uint(s[4 * n + 1]),
                 __float_as_uint(s[4 * n + 2]), __float_as_uint(s[4 * n + 3])};
  }
  static __device__ __forceinline__ float sum(u32x4 w, float acc) {
    return acc + ((__uint_as_float(w[0]) + __uint_as_float(w[1])) +
                  (__uint_as_float(w[2]) + __uint_as_float(w[3])));
  }
};

// Layout of an LDS tile: rows of D elements without padding, 16-byte chunk c of
// row r at chunk position c ^ swz(r).  Tiles are read by rows (16 bytes of each
// of 16 rows per cycle) and by columns (the k operand transposed).
//   16-bit: as the backward's tiles in attn_bwd.hip (bwd_swz): conflict-free row
//     reads, the transposing read's four rows on different banks;
//   fp32: r & 15, a 256-byte bank line holds a row or half of one.  The column
//     reads take 32 consecutive elements of one row and have no conflicts anyway.
template <typename E, int D>
struct Lay {
  static constexpr int ESZ = Elem<E>::kBytes;
  static constexpr int KCH = 16 / ESZ;      // elements per chunk
  static constexpr int RB = D * ESZ;        // bytes per row
  static constexpr int CPR = RB / 16;       // chunks per row
  static constexpr int RPS = 64 / CPR;      // rows per 1 KB slice (one wave instruction)
  static constexpr int KS = CPR / 2;        // chunk steps over the head dim
  static constexpr int DB = D / 32;         // 32-column blocks
  static constexpr int NG = Elem<E>::kGroups;
  static __device__ __forceinline__ int swz(int r) {
    if constexpr (ESZ == 4) return r & 15;
    const int s = ((r & 3) << 1) | ((r >> 2) & 1);
    return CPR == 8 ? s ^ (((r >> 3) & 1) << 1) : s | (((r >> 3) & 1) << 3);
  }
};

// A lane's byte offsets for both kinds of read (row l32 = lane % 32, half g).
// refresh() keeps the compiler from folding a buffer's base into a register for
// each of them.
template <typename E, int D>
struct Reads {
  using L = Lay<E, D>;
  static constexpr int NR = L::KS < 8 ? L::KS : 8;          // beyond: + 256 bytes
  static constexpr int NT = L::ESZ == 4 ? 4 : 2 * L::DB;
  int r[NR], t[NT];
  // `block`: the 32-row block that block 0 below stands for.
  __device__ __forceinline__ void init(int lane, int block = 0) {
    const int l32 = lane & 31, g = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < NR; ++ks) r[ks] = l32 * L::RB + (((2 * ks + g) ^ L::swz(l32)) << 4);
    if constexpr (L::ESZ == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        t[i] = (4 * g + i) * L::RB + ((((l32 >> 2) ^ (4 * g)) ^ i) << 4) + 4 * (l32 & 3);
    } else {
      const int row = 4 * g + ((lane & 15) >> 2);
      const int ch = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
      for (int db = 0; db < L::DB; ++db)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          t[2 * db + h] = (row + 8 * h) * L::RB + (((4 * db + ch) ^ L::swz(row + 8 * h)) << 4) +
                          8 * (lane & 1);
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) r[i] += 32 * block * L::RB;
#pragma unroll
    for (int i = 0; i < NT; ++i) t[i] += 32 * block * L::RB;
  }
  __device__ __forceinline__ void refresh() {
#pragma unroll
    for (int i = 0; i < NR; ++i) opaque(r[i]);
#pragma unroll
    for (int i = 0; i < NT; ++i) opaque(t[i]);
  }
  // Chunk 2 ks + g of row l32 of 32-row block kb.
  __device__ __forceinline__ u32x4 row(const char* tile, int kb, int ks) const {
    return *(const u32x4*)(tile + 32 * kb * L::RB + 256 * (ks / NR) + r[ks % NR]);
  }
  // Column 32 db + l32 of the rows of k-group n of block kb.
  __device__ __forceinline__ u32x4 col(const char* tile, int kb, int n, int db) const {
    if constexpr (L::ESZ == 4) {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = *(const uint32_t*)(tile + (32 * kb + 8 * n) * L::RB + 128 * (db ^ (n & 1)) + t[i]);
      return w;
    } else {
      const char* p = tile + (32 * kb + 16 * n) * L::RB;
      const u32x2 lo = ds_read_tr16((const uint16_t*)(p + t[2 * db]));
      const u32x2 hi = ds_read_tr16((const uint16_t*)(p + t[2 * db + 1]));
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
  }
};

// Fills ROWS-row tiles from a [rows, D] tensor with direct global -> LDS loads:
// wave w fills slices w, w + NW, ...  Chunks at or past the tensor's head dim
// and rows at or past `rows` arrive as zeros.
// AUX: cache policy of the loads (0, or kOnce for what nothing reads again).
constexpr int kOnce = 2;  // non-temporal
template <int AUX>
__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t rs, uint32_t off, char* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 16,
                                           off, 0, 0, AUX);
}
template <typename E, int D, int ROWS, int NW = 4, int AUX = 0>
struct Stage {
  using L = Lay<E, D>;
  static constexpr int SPW = ROWS * L::RB / 1024 / NW;
  static_assert(SPW >= 1, "a slice per wave");
  const char* base;
  int64_t sb;          // bytes per row
  uint32_t off[SPW];
  uint32_t tail;       // bytes of the last row
  __device__ __forceinline__ void init(const TensorArg& t, int b, int h, int dch, int lane,
                                       int wave) {
    base = (const char*)t.ptr + (b * t.sb + h * t.sh) * L::ESZ;
    sb = t.ss * L::ESZ;
    tail = 16u * dch;
#pragma unroll
    for (int m = 0; m < SPW; ++m) {
      const int r = row(m, lane, wave);
      const int ch = (lane % L::CPR) ^ L::swz(r);
      off[m] = ch >= dch ? kOobOffset : (uint32_t)(r * (int)sb + 16 * ch);
    }
  }
  static __device__ __forceinline__ int row(int m, int lane, int wave) {
    return (wave + NW * m) * L::RPS + lane / L::CPR;
  }
  // Rows [row0, row0 + ROWS), those at or past n as zeros.
  __device__ __forceinline__ void load(int row0, int n, char* tile, int wave) const {
    const int rows = min(ROWS, n - row0);
    const auto rs = tile_rsrc(base + row0 * sb, (uint32_t)((rows - 1) * (int)sb) + tail);
#pragma unroll
    for (int m = 0; m < SPW; ++m)
      load_lds16<AUX>(rs, off[m], tile + (wave + NW * m) * 1024);
  }
  // The same with rows of negative document id as zeros too (their contents may
  // be anything, and 0 * NaN is not 0).  ids: of row row0 and on.
  __device__ __forceinline__ void load_padded(int row0, int n, char* tile, int lane, int wave,
                                              const int* ids) const {
    const int rows = min(ROWS, n - row0);
    const auto rs = tile_rsrc(base + row0 * sb, (uint32_t)((rows - 1) * (int)sb) + tail);
    uint32_t o[SPW];
#pragma unroll
    for (int m = 0; m < SPW; ++m) {
      const int r = row(m, lane, wave);
      o[m] = r < rows && ids[r] >= 0 ? off[m] : kOobOffset;
    }
#pragma unroll
    for (int m = 0; m < SPW; ++m)
      load_lds16<AUX>(rs, o[m], tile + (wave + NW * m) * 1024);
  }
};

// Scores in log2 units: x = f * y + b0 - slope2 * |i - j| of y, the raw product s or
// what the cap makes of it.
struct ScoreConst {
  float f, b0;
  float k1;  // cap: 2 * log2(e) * scale / cap
  float kz;  // cap: scale / cap
};

// y with a cap: tanh(z) = 1 - 2 / (1 + exp(2 z)).
//   16-bit inputs: y = -1 / (1 + exp(2 z)), f = 2 cap log2(e), b0 = cap log2(e): one
//   multiply-add fewer per score.  Off by about 1e-7 absolutely, cap * 1e-7 in the
//   score, far below the rounding of P.
//   fp32: y = tanh(z), f = cap log2(e), b0 = 0, by the Taylor series below |z| = 0.4
//   (7 terms, the next one 4e-9), where the formula loses the leading digits.
template <typename E, bool CAP>
__device__ __forceinline__ float score_y(float s, const ScoreConst& k) {
  if constexpr (!CAP) {
    return s;
  } else if constexpr (Elem<E>::kBytes == 2) {
    return __builtin_amdgcn_rcpf(-1.f - fast_exp2(s * k.k1));
  } else {
    const float t =
        __builtin_fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + fast_exp2(s * k.k1)), 1.f);
    const float z = s * k.kz, u = z * z;
    float p = __builtin_fmaf(u, 21844.f / 6081075.f, -1382.f / 155925.f);
    p = __builtin_fmaf(u, p, 62.f / 2835.f);
    p = __builtin_fmaf(u, p, -17.f / 315.f);
    p = __builtin_fmaf(u, p, 2.f / 15.f);
    p = __builtin_fmaf(u, p, -1.f / 3.f);
    p = __builtin_fmaf(u * p, z, z);
    return u < 0.16f ? p : t;
  }
}
// d score / d raw product, over scale: 1 - tanh^2.
template <typename E, bool CAP>
__device__ __forceinline__ float score_slope(float y) {
  if constexpr (!CAP) return 1.f;
  else if constexpr (Elem<E>::kBytes == 2) return -4.f * y * (y + 1.f);
  else return __builtin_fmaf(-y, y, 1.f);
}

// What 64 rows' document ids say: range of the ids >= 0 (lo > hi: none), whether
// any is negative.  One record per 64 keys, then one per 64 queries.
struct DocTile {
  int lo, hi, pad, unused;
};

struct SAttnArgs {
  TensorArg q, k, v, o, dout, dq, dk, dv;
  float* lse;
  const float* delta;
  const float* lse2;
  const float* slopes;
  const int* docs;       // [B, Sk]
  const int* prefix;     // [B]
  const DocTile* ktiles; // [B, ceil(Sk / 64)]
  const DocTile* qtiles; // [B, ceil(Sq / 64)]
  int B, H, Hk, G, Sq, Sk, D;
  int off;               // Sk - Sq: position of query 0
  int dch;               // 16-byte chunks of D
  int causal;
  float scale;
  ScoreConst sc;
  // Sums split over several workgroups ("parts"), joined by a second launch: O of a
  // query tile (forward), dK / dV of a key tile and dQ of a query tile (backward).
  int parts, qparts;     // forward: parts; backward: parts of dK / dV, of dQ
  float *part, *qpart;   // accumulators as they lie, see part_at
  float* ml;             // forward: reference and sum of each part's rows
  void* olo;             // forward: O - round(O), strides of o, or null
};

// One new token of each sequence over its cache (decode.hip).
struct DecodeArgs {
  const void* q;
  void* o;
  int64_t q_sb, q_sh, o_sb, o_sh;
  TensorArg k, v;
  const float* slopes;
  const int* lengths;  // [B] or null: S keys each
  int B, H, Hk, G, S, D, dch, splits;
  ScoreConst sc;
  float* part;         // [B * H, splits, D]
  float* ml;           // [B * H, splits, 2]
};

// Document ids of up to 128 rows, by blocks of 32, seen by a whole wave: block i's range
// in the lanes from kBlockLane[i] on (eight scalars would be spilled for the length of
// a kernel that needs them now and then); bit i of pad: a negative id in block i.
struct DocRange {
  int lo, hi, pad;
  static constexpr int kBlockLane[4] = {0, 32, 16, 48};
  __device__ __forceinline__ int block_lo(int i) const {
    return __builtin_amdgcn_readlane(lo, kBlockLane[i]);
  }
  __device__ __forceinline__ int block_hi(int i) const {
    return __builtin_amdgcn_readlane(hi, kBlockLane[i]);
  }
};
__device__ __forceinline__ DocRange doc_range(const int* ids, int row0, int n, int lane) {
  int lo[2], hi[2], pad = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = lane + 64 * j, d = i < n ? ids[row0 + i] : 0x7fffffff;
    const bool some = i < n && d >= 0;
    lo[j] = some ? d : 0x7fffffff;
    hi[j] = some ? d : -1;
#pragma unroll
    for (int m = 16; m; m >>= 1) {
      lo[j] = min(lo[j], __shfl_xor(lo[j], m, 64));
      hi[j] = max(hi[j], __shfl_xor(hi[j], m, 64));
    }
    const uint64_t p = __ballot(d < 0);
    pad |= ((uint32_t)p ? 1 << 2 * j : 0) | (p >> 32 ? 2 << 2 * j : 0);
  }
  const bool second = lane & 16;
  return {second ? lo[1] : lo[0], second ? hi[1] : hi[0], pad};
}

// The streamed tiles a workgroup has to visit, in order.  Without documents a range;
// with them a list in LDS, built 64 tiles at a time (lane t looks at one tile, a
// ballot gives the live ones their places), at most kListed tiles of the sequence in
// one list.  An entry is a tile's index; for each block of 32 of the workgroup's rows
// kLive (it shares a document with the tile: the others' waves have nothing to do)
// and kFull (every pair visible: no mask); and kPad (rows of negative document id in
// it).  The walk over it, `heads` times for dK / dV, takes the entries part,
// part + parts, ...: equal shares whatever the mask.
constexpr int kTileIndex = (1 << 20) - 1, kFull = 1 << 20, kLive = 1 << 24, kPad = 1 << 29;
constexpr int kBlocks = 15;  // all four of either
constexpr int kListed = 512;

// kLive, kPad and, as far as documents go, kFull of a tile.
__device__ __forceinline__ int doc_bits(const DocTile& w, const DocRange& own) {
  int f = w.pad ? kPad : 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int lo = own.block_lo(i), hi = own.block_hi(i);
    if (w.lo <= hi && w.hi >= lo) f |= kLive << i;
    if (w.lo == w.hi && w.lo == lo && w.lo == hi && !w.pad && !(own.pad >> i & 1))
      f |= kFull << i;
  }
  return f;
}

struct TileWalk {
  const int* list;                 // null: tiles [lo, lo + count), full in [f0, f1)
  int lo, f0, f1;
  int count, at, parts, head, hend;
  __device__ __forceinline__ int entry() const {  // -1 behind the last
    if (head >= hend) return -1;
    if (list) return __builtin_amdgcn_readfirstlane(list[at]);
    const int t = lo + at;
    return t | kLive * kBlocks | (t >= f0 && t < f1 ? kFull * kBlocks : 0);
  }
  __device__ __forceinline__ void step(int n) {
    at += n;
    while (at >= count && head < hend) {
      at -= count;
      ++head;
    }
  }
  __device__ __forceinline__ void begin(int part, int parts_, int head_, int heads) {
    at = 0;
    parts = parts_;
    hend = head_ + heads;
    head = count > 0 ? head_ : hend;
    step(part);
  }
};

// Tiles [first, first + kListed) of n; `look` gives an entry's bits, kLive for none if
// the tile is not visited.
// Ends with a barrier.
template <typename F>
__device__ __forceinline__ int tile_list(int* list, int first, int n, F look) {
  const int lane = threadIdx.x & 63, end = min(n, first + kListed);
  int count = 0;
  for (int t0 = first; t0 < end; t0 += 64) {
    const int f = t0 + lane < end ? look(t0 + lane) : 0;
    const uint64_t live = __ballot(f & kLive * kBlocks);
    if ((f & kLive * kBlocks) && threadIdx.x < 64)
      list[count + __popcll(live & ((1ull << lane) - 1))] = (t0 + lane) | f;
    count += __popcll(live);
  }
  __syncthreads();
  return count;
}

// A part's accumulators (32 rows, DB column blocks) in the workspace, as they lie in
// the registers: whole 1 KB stores and loads.  `index`: which rows, tensor and part.
template <int DB>
__device__ __forceinline__ f32x4* part_at(float* part, int64_t index) {
  return (f32x4*)(part + index * (DB * 1024));
}
template <int DB>
__device__ __forceinline__ void part_store(const f32x16 (&acc)[DB], f32x4* p, int lane) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int jj = 0; jj < 4; ++jj)
      p[(4 * db + jj) * 64 + lane] = f32x4{acc[db][4 * jj], acc[db][4 * jj + 1],
                                           acc[db][4 * jj + 2], acc[db][4 * jj + 3]};
}
// acc += w * the part
template <int DB>
__device__ __forceinline__ void part_add(f32x16 (&acc)[DB], const f32x4* p, int lane, float w) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
      const f32x4 x = p[(4 * db + jj) * 64 + lane];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[db][4 * jj + i] = __builtin_fmaf(x[i], w, acc[db][4 * jj + i]);
    }
}

// Writes one wave's 32 x D block, held transposed in 32x32 accumulators, times a
// per-lane factor, rounded to E: staged through the wave's own LDS region (32
// rows) so that each lane stores 16 contiguous bytes.  Chunks at or past dch and
// rows at or past nrows are not stored.
// LO (16-bit types): what the rounding to E leaves, rounded to E, instead.
template <typename E, int D, bool LO = false>
__device__ __forceinline__ void store_rows(const f32x16 (&acc)[D / 32], float sc, char* lds,
                                           char* out, int64_t row_bytes, int dch, int nrows) {
  using L = Lay<E, D>;
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
      const float a = acc[db][4 * jj] * sc, b = acc[db][4 * jj + 1] * sc,
                  c = acc[db][4 * jj + 2] * sc, d = acc[db][4 * jj + 3] * sc;
      if constexpr (L::ESZ == 4) {
        const int ch = 8 * db + 2 * jj + g;
        *(f32x4*)(lds + l32 * L::RB + ((ch ^ (l32 & 7)) << 4)) = f32x4{a, b, c, d};
      } else {
        const int ch = 4 * db + jj;
        u32x2 w = Elem<E>::pack4(a, b, c, d);
        if constexpr (LO)
          w = Elem<E>::pack4(a - E::to_f32(w[0] & 0xffff), b - E::to_f32(w[0] >> 16),
                             c - E::to_f32(w[1] & 0xffff), d - E::to_f32(w[1] >> 16));
        *(u32x2*)(lds + l32 * L::RB + ((ch ^ (l32 & 7)) << 4) + 8 * g) = w;
      }
    }
#pragma unroll
  for (int p = 0; p < 32 / L::RPS; ++p) {
    const int r = p * L::RPS + lane / L::CPR, ch = lane % L::CPR;
    const u32x4 w = *(const u32x4*)(lds + r * L::RB + ((ch ^ (r & 7)) << 4));
    if (ch < dch && r < nrows)
      __builtin_nontemporal_store(w, (u32x4*)(out + r * row_bytes + 16 * ch));
  }
}

}  // namespace mi
