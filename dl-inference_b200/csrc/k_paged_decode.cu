// Attention of few new tokens over a paged KV cache (decode steps, short
// speculative runs; float32 calls of any length): tensor cores by mma.sync, K/V
// pages by TMA, 16-bit, float32 or 4-bit pages, head dims 64 and 128.
//
// A unit is one row tile (8 or 16 query rows: the new tokens of a sequence times
// the query heads of one KV head) over all its visible keys. S^T = K Q^T puts 16
// keys on the m16 side and the rows on n8, O^T = V^T P^T likewise, so 7 heads
// waste an eighth of the tensor work; each K/V byte is fetched once per tile.
//
// The work of a call is the list of all key blocks of all units, in order; CTA c
// of G takes the c-th of G equal shares of it, whatever the sequences' lengths
// are (a ragged batch keeps every SM busy to the end). A unit that lies within
// one share is finished there; of the others each CTA stores its part's (max,
// sum, O) in the workspace and a second kernel merges the parts in order
// (deterministic). A call whose units cannot be long runs one CTA per unit and
// needs no merge.
//
// One producer warp walks the page table and issues the TMA boxes of each block
// (a page's rows of one head; boxes past the sequence or of a bad page read as
// zeros), K and V as entries of one ring; the consumer warps take 16 keys of the
// block each. Every wait is bounded.
//
// 4-bit pages: a (page, head) block is contiguous and arrives by one untiled bulk
// copy (tiled boxes of 64- and 16-byte rows held the TMA at 3.8 TB/s); codes
// become halves in registers, in the order of the MMA fragments: E2M1 x E4M3 has 6 significant bits, so the
// products are exact, and the MMA runs in f16 for every model type. q is scaled for that
// by a power of two per row, its largest element to [1, 2): a half keeps all 11 bits of
// elements down to 2^-14, smaller ones to 2^-25 of the row's maximum; a float32 q, and
// its P, enter as two halves each (22 bits).
//
// P is rounded to the model's 16-bit type for its product with V (to halves over 4-bit
// pages), sums and O stay in fp32: the error against 64 bits of a bf16 output is 2.1e-3
// where its own rounding alone gives 1.7e-3, of f16 2.7e-4 and 2.1e-4. The exponentials
// are ex2.approx (2^-22), the cap's reciprocal rcp.approx (2^-23).
//
// float32 pages: every operand is split into two TF32 numbers and three of the four
// products are summed (2^-22 relative; 2.4e-7 against 64 bits in all), so the call stays bound
// by memory instead of by FFMA. MMAs cut their sums off, which would bias long
// chains: scores are summed in four, O in one per 16 keys, and added up in fp32.
//
// Bound by memory when the cache is long (3 sequences of up to 60001 keys, 64/8 heads of
// 128: 102 us = 6.1 TB/s), by its start, the second kernel and the ragged ends when it is
// not (32 x up to 2304 keys, 28/4 heads: 26.7 us = 4.2 TB/s; 1 x 333 keys 6 us). 4-bit
// pages: the conversion (24 x up to 8192 keys, 28/4 heads: 34 us; ALU 51% busy, issue 57%
// with 12 consumer warps per SM; eight per CTA spilled). float32: 32 x up to 1501 keys,
// 16/4 heads: 40 us = 3.6 TB/s (ALU 38%, issue 40% busy); prompts in tiles of 8 rows, for
// each of which K and V are fetched and split again: 4 x 512 tokens, 16/4 heads, 380 us.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <map>
#include <mutex>
#include <type_traits>
#include <utility>

#include "mma_sync.cuh"
#include "paged_attn.cuh"
#include "tcgen05.cuh"

namespace dli_sm100 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
struct DecodeArgs {
  PagedAttnArgs a;
  int tiles_max;   // row tiles of a sequence of max_new tokens
  int split;       // 0: one CTA per unit
  int min_blocks;  // split: the shares are no smaller, with fewer CTAs at work
  int ctas;        // split: CTAs of the main kernel
  float* part_o;   // [2 ctas][rows][D]
  float2* part_ml; // [2 ctas][rows]: running maximum (log2) and sum
};

// W consumer warps: 4, or 8 where the ring's entries are small enough. Two CTAs per
// SM, one works while the other waits (float32, 32 x 1501 keys, 16/4 heads: one CTA of 8
// warps took a tenth longer than two of 4, although a few registers spill);
// 4-bit pages three, or one with two row tiles or split float32 operands.
template <typename T, typename KV, int D, int NT>
struct DecodeLayout {
  static constexpr bool kFp4 = std::is_same<KV, Fp4>::value;
  static constexpr bool kF32 = std::is_same<KV, float>::value;
  static constexpr int W = !kFp4 && !kF32 && D == 64 && NT == 1 ? 8 : 4;
  static constexpr int SUB = kFp4 ? 2 : 1;  // 16-key groups of a warp per block
  static constexpr int kThreads = 32 * W + 32;
  static constexpr int R = 8 * NT;
  static constexpr int BN = 16 * W * SUB;  // keys per block
  static constexpr int kCtas = kFp4 && (NT == 2 || std::is_same<T, float>::value) ? 1 : kFp4 ? 3 : 2;
  static constexpr int kRowBytes = kFp4 ? D / 2 : kF32 ? D * 4 : D * 2;
  static constexpr int kBox = BN * 128;          // bytes of one 128-byte-wide column of boxes
  static constexpr int kCodes = BN * kRowBytes;  // code or element bytes of a K (or V) block
  static constexpr int kEntry = kCodes + (kFp4 ? BN * D / 16 : 0);
  static constexpr int DH = 64;  // dims that the warps merge at a time
  static constexpr int kMerge = W * R * DH * 4;
  static constexpr int kMl = 2 * W * R * 4;
  static constexpr int kRoom = (kCtas == 3 ? 75 : kCtas == 2 ? 113 : 227) * 1024 - kMerge - kMl - 1024 - 256;
  static constexpr int kEntries = (kRoom / kEntry) < 16 ? (kRoom / kEntry) : 16;
  static constexpr int kMergeOff = kEntries * kEntry;
  static constexpr int kMlOff = kMergeOff + kMerge;
  static constexpr int kBarOff = kMlOff + kMl;
  static constexpr int kBytes = kBarOff + 2 * kEntries * 8 + 1024;  // the ring's base is rounded up to 1 KiB
  static_assert(kEntry % (kFp4 ? 16 : 1024) == 0, "entry alignment");
  static_assert(kEntries >= 3, "a ring that overlaps loads with work");
  static_assert(kBytes <= 232448, "shared memory");
};

// What one sequence contributes to the list of key blocks.
struct SeqWork {
  SeqRows rows;
  int tiles, blocks, block0, kv_len, key_lo;
};

template <int BN, int R>
__device__ __forceinline__ SeqWork seq_work(const PagedAttnArgs& a, int b, bool report) {
  SeqWork w;
  w.rows = seq_rows(a.seqs, b, report);
  w.kv_len = w.rows.past + w.rows.n;
  w.key_lo = a.window <= w.rows.past ? w.rows.past - a.window + 1 : 0;
  w.tiles = (w.rows.n * a.group + R - 1) / R;
  w.block0 = w.key_lo / BN;
  w.blocks = (w.kv_len + BN - 1) / BN - w.block0;
  return w;
}

// The equal shares of `total` blocks among the CTAs that get any.
struct Shares {
  int total, ctas, q, r;
  __device__ __forceinline__ Shares(int total_blocks, int grid, int min_blocks) : total(total_blocks) {
    ctas = max(1, min(grid, (total + min_blocks - 1) / min_blocks));
    q = total / ctas;
    r = total - q * ctas;
  }
  __device__ __forceinline__ int begin(int c) const { return c >= ctas ? total : c * q + min(c, r); }
  __device__ __forceinline__ int cta_of(int at) const { return at < r * (q + 1) ? at / (q + 1) : r + (at - r * (q + 1)) / max(q, 1); }
};

// The blocks of all sequences (a whole warp).
template <int BN, int R>
__device__ __forceinline__ int list_total(const PagedAttnArgs& a, int lane, bool report) {
  int total = 0;
  for (int c = 0; c < a.seqs.batch; c += 32) {
    if (c + lane < a.seqs.batch) {
      const SeqWork s = seq_work<BN, R>(a, c + lane, report);
      total += a.hkv * s.tiles * s.blocks;
    }
  }
  return __reduce_add_sync(0xffffffffu, total);
}

struct Segment {
  int b, kvh, rt, block, blocks;  // key blocks [block, block + blocks) of the unit
  bool whole;
  int slot;  // of the part, when not whole
  SeqWork w;
};

// Walks the segments of a CTA's share; every warp runs its own copy.
template <int BN, int R>
struct Walker {
  const DecodeArgs& d;
  int w, w_end, w0, base, work, b;
  SeqWork sw;

  __device__ __forceinline__ void take(int seq) {
    b = seq;
    sw = seq_work<BN, R>(d.a, seq, false);
    work = d.a.hkv * sw.tiles * sw.blocks;
  }

  __device__ Walker(const DecodeArgs& args, int lane) : d(args) {
    base = b = work = 0;
    if (!d.split) {
      w = 0;
      w_end = 1;
      return;
    }
    const int total = list_total<BN, R>(d.a, lane, blockIdx.x == 0);
    const Shares shares(total, d.ctas, d.min_blocks);
    w0 = w = shares.begin(blockIdx.x);
    w_end = shares.begin(blockIdx.x + 1);
    if (w >= w_end) return;
    // the sequence that holds w (the loads are the first pass's: they hit L1)
    const int batch = d.a.seqs.batch;
    for (int c = 0; c < batch; c += 32) {
      int mine = 0;
      if (c + lane < batch) {
        const SeqWork s = seq_work<BN, R>(d.a, c + lane, false);
        mine = d.a.hkv * s.tiles * s.blocks;
      }
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const int k = __popc(__ballot_sync(0xffffffffu, base + upto <= w));  // sequences that end before w
      if (k < 32) {
        base += __shfl_sync(0xffffffffu, upto - mine, k);
        take(c + k);
        return;
      }
      base += __shfl_sync(0xffffffffu, upto, 31);
    }
  }

  __device__ bool get(Segment& s) {
    if (w >= w_end) return false;
    if (!d.split) {
      w = w_end;
      const int per = d.a.hkv * d.tiles_max;
      s.b = blockIdx.x / per;
      const int u = blockIdx.x - s.b * per;
      s.kvh = u / d.tiles_max;
      s.rt = u - s.kvh * d.tiles_max;
      s.w = seq_work<BN, R>(d.a, s.b, u == 0);
      if (s.rt >= s.w.tiles) return false;
      s.block = s.w.block0;
      s.blocks = s.w.blocks;
      s.whole = true;
      s.slot = 0;
      return true;
    }
    while (w >= base + work) {
      base += work;
      take(b + 1);
    }
    const int rel = w - base;
    const int unit = rel / sw.blocks, blk = rel - unit * sw.blocks;
    s.b = b;
    s.kvh = unit / sw.tiles;
    s.rt = unit - s.kvh * sw.tiles;
    s.w = sw;
    s.block = sw.block0 + blk;
    s.blocks = min(sw.blocks - blk, w_end - w);
    s.whole = s.blocks == sw.blocks;
    s.slot = 2 * blockIdx.x + (w == w0 ? 0 : 1);
    w += s.blocks;
    return true;
  }
};

// Four output values as T.
template <typename T>
__device__ __forceinline__ void store4(T* dst, float x, float y, float z, float w) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = make_float4(x, y, z, w);
  else *reinterpret_cast<uint2*>(dst) = make_uint2(pack16<T>(x, y), pack16<T>(z, w));
}

// Byte offset of (key row, 16-bit column) in a K or V block of columns of `box` bytes:
// [keys][64 elements] with the 128-byte swizzle.
__device__ __forceinline__ int swz128(int box, int row, int col) {
  return (col >> 6) * box + row * 128 + ((((col >> 3) & 7) ^ (row & 7)) << 4) + (col & 7) * 2;
}

// ---- the two products of 16 keys: S^T = K Q^T (sc is written) and O^T += V^T P^T
// (sc holds p). sc[nt][i]: key row g (+ 8 for i >= 2), query row nt * 8 + 2t + (i & 1).

template <typename T, int D, int NT>
__device__ __forceinline__ void qk_16(float (&sc)[NT][4], uint32_t k, int box, int kw, int lane,
                                      const uint32_t (&qf)[NT][D / 16][2]) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    uint32_t f[4];
    ldmatrix_x4(f, k + swz128(box, kw + (lane & 15), kk * 16 + (lane >> 4) * 8));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) mma_16816<T>(sc[nt], f[0], f[1], f[2], f[3], qf[nt][kk][0], qf[nt][kk][1]);
  }
}
template <typename T, int D, int NT>
__device__ __forceinline__ void pv_16(float (&o)[NT][D / 16][4], const float (&p)[NT][4], uint32_t v, int box, int kw, int lane) {
  uint32_t pb[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    pb[nt][0] = movmatrix_trans(pack16<T>(p[nt][0], p[nt][1]));
    pb[nt][1] = movmatrix_trans(pack16<T>(p[nt][2], p[nt][3]));
  }
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    uint32_t f[4];
    ldmatrix_x4_trans(f, v + swz128(box, kw + (lane & 7) + (lane >> 4) * 8, i * 16 + ((lane >> 3) & 1) * 8));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) mma_16816<T>(o[nt][i], f[0], f[1], f[2], f[3], pb[nt][0], pb[nt][1]);
  }
}

// float32: K rows perm(g), perm(g) + 8 by 16 bytes, 4 dims of each 16.
template <int D, int NT>
__device__ __forceinline__ void qk_f32(float (&sc)[NT][4], const uint8_t* sk, int box, int kw, int g, int t,
                                       const uint32_t (&qf)[NT][D / 16][4]) {
  const int r0 = kw + ((g >> 1) | ((g & 1) << 2)), r1 = r0 + 8;
  float part[NT][4][4], low[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i) low[nt][i] = part[nt][0][i] = part[nt][1][i] = part[nt][2][i] = part[nt][3][i] = 0.f;
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const uint8_t* col = sk + (kk >> 1) * box;
    const int ch = (kk & 1) * 4 + t;
    const float4 k0 = *reinterpret_cast<const float4*>(col + r0 * 128 + ((ch ^ (r0 & 7)) << 4));
    const float4 k1 = *reinterpret_cast<const float4*>(col + r1 * 128 + ((ch ^ (r1 & 7)) << 4));
    uint32_t hi[2][4], lo[2][4];
    split_tf32<true>(k0.x, hi[0][0], lo[0][0]);
    split_tf32<true>(k1.x, hi[0][1], lo[0][1]);
    split_tf32<true>(k0.y, hi[0][2], lo[0][2]);
    split_tf32<true>(k1.y, hi[0][3], lo[0][3]);
    split_tf32<true>(k0.z, hi[1][0], lo[1][0]);
    split_tf32<true>(k1.z, hi[1][1], lo[1][1]);
    split_tf32<true>(k0.w, hi[1][2], lo[1][2]);
    split_tf32<true>(k1.w, hi[1][3], lo[1][3]);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float(&acc)[4] = part[nt][kk & 3];
      mma_1688_f32(acc, low[nt], hi[0], lo[0], __uint_as_float(qf[nt][kk][0]), __uint_as_float(qf[nt][kk][1]));
      mma_1688_f32(acc, low[nt], hi[1], lo[1], __uint_as_float(qf[nt][kk][2]), __uint_as_float(qf[nt][kk][3]));
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      sc[nt][i] = low[nt][i] + ((part[nt][0][i] + part[nt][1][i]) + (part[nt][2][i] + part[nt][3][i]));
}
// V: the 4 dims of 16-byte chunk c(g) of each 32, of the keys perm(2t) = t and
// perm(2t + 1) = t + 4 of each 8.
__device__ __forceinline__ int f32_chunk(int g) { return ((g & 1) << 2) | (g >> 1); }
template <int D, int NT>
__device__ __forceinline__ void pv_f32(float (&o)[NT][D / 16][4], const float (&p)[NT][4], const uint8_t* sv, int box, int kw,
                                       int g, int t) {
  float pb[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    // P^T as the B operand: lane (g, t) gets rows g of the keys 2t, 2t + 1 (+ 8)
    const int s0 = 8 * t + (g >> 1), s1 = s0 + 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float x0 = __shfl_sync(0xffffffffu, p[nt][2 * h], s0), y0 = __shfl_sync(0xffffffffu, p[nt][2 * h + 1], s0);
      const float x1 = __shfl_sync(0xffffffffu, p[nt][2 * h], s1), y1 = __shfl_sync(0xffffffffu, p[nt][2 * h + 1], s1);
      pb[nt][2 * h] = (g & 1) ? y0 : x0;
      pb[nt][2 * h + 1] = (g & 1) ? y1 : x1;
    }
  }
  const int chunk = f32_chunk(g);
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const uint8_t* col = sv + i * box;
    float part[NT][2][4], low[NT][2][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 4; ++k) part[nt][0][k] = part[nt][1][k] = low[nt][0][k] = low[nt][1][k] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int ra = kw + h * 8 + t, rb = ra + 4;
      const float4 va = *reinterpret_cast<const float4*>(col + ra * 128 + ((chunk ^ (ra & 7)) << 4));
      const float4 vb = *reinterpret_cast<const float4*>(col + rb * 128 + ((chunk ^ (rb & 7)) << 4));
      uint32_t hi[2][4], lo[2][4];
      split_tf32<true>(va.x, hi[0][0], lo[0][0]);
      split_tf32<true>(va.y, hi[0][1], lo[0][1]);
      split_tf32<true>(vb.x, hi[0][2], lo[0][2]);
      split_tf32<true>(vb.y, hi[0][3], lo[0][3]);
      split_tf32<true>(va.z, hi[1][0], lo[1][0]);
      split_tf32<true>(va.w, hi[1][1], lo[1][1]);
      split_tf32<true>(vb.z, hi[1][2], lo[1][2]);
      split_tf32<true>(vb.w, hi[1][3], lo[1][3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma_1688_f32(part[nt][0], low[nt][0], hi[0], lo[0], pb[nt][2 * h], pb[nt][2 * h + 1]);
        mma_1688_f32(part[nt][1], low[nt][1], hi[1], lo[1], pb[nt][2 * h], pb[nt][2 * h + 1]);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        o[nt][2 * i][k] += part[nt][0][k] + low[nt][0][k];
        o[nt][2 * i + 1][k] += part[nt][1][k] + low[nt][1][k];
      }
  }
}

// 4-bit: code and scale are this thread's places in key row perm(g); dims t * D/4 ..
// in the order of the code bytes.
template <int D, int NT, int QS>
__device__ __forceinline__ void qk_fp4(float (&sc)[NT][4], const uint8_t* code, const uint8_t* scale,
                                       const uint32_t (&qf)[NT][D / 16][2 * QS]) {
  uint32_t w0[D / 32], w1[D / 32], s0[D / 64], s1[D / 64];
  if constexpr (D == 128) {
    const uint4 c0 = *reinterpret_cast<const uint4*>(code), c1 = *reinterpret_cast<const uint4*>(code + 8 * 64);
    w0[0] = c0.x, w0[1] = c0.y, w0[2] = c0.z, w0[3] = c0.w;
    w1[0] = c1.x, w1[1] = c1.y, w1[2] = c1.z, w1[3] = c1.w;
    const uint32_t e0 = e4m3x2_to_half2(*reinterpret_cast<const uint16_t*>(scale));
    const uint32_t e1 = e4m3x2_to_half2(*reinterpret_cast<const uint16_t*>(scale + 8 * 8));
    s0[0] = __byte_perm(e0, e0, 0x1010), s0[1] = __byte_perm(e0, e0, 0x3232);
    s1[0] = __byte_perm(e1, e1, 0x1010), s1[1] = __byte_perm(e1, e1, 0x3232);
  } else {
    const uint2 c0 = *reinterpret_cast<const uint2*>(code), c1 = *reinterpret_cast<const uint2*>(code + 8 * 32);
    w0[0] = c0.x, w0[1] = c0.y;
    w1[0] = c1.x, w1[1] = c1.y;
    const uint32_t e = e4m3x2_to_half2(static_cast<uint32_t>(scale[0]) | (static_cast<uint32_t>(scale[8 * 4]) << 8));
    s0[0] = __byte_perm(e, e, 0x1010);
    s1[0] = __byte_perm(e, e, 0x3232);
  }
  float part[NT][2][4];  // two chains
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int k = 0; k < 4; ++k) part[nt][0][k] = part[nt][1][k] = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {  // a code word: two MMAs
    const uint32_t x0 = s0[i / 2], x1 = s1[i / 2];
    const uint32_t a00 = mul_half2(e2m1x2_to_half2<0>(w0[i]), x0), a01 = mul_half2(e2m1x2_to_half2<1>(w0[i]), x0);
    const uint32_t a02 = mul_half2(e2m1x2_to_half2<2>(w0[i]), x0), a03 = mul_half2(e2m1x2_to_half2<3>(w0[i]), x0);
    const uint32_t a10 = mul_half2(e2m1x2_to_half2<0>(w1[i]), x1), a11 = mul_half2(e2m1x2_to_half2<1>(w1[i]), x1);
    const uint32_t a12 = mul_half2(e2m1x2_to_half2<2>(w1[i]), x1), a13 = mul_half2(e2m1x2_to_half2<3>(w1[i]), x1);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = QS - 1; k >= 0; --k) {
        mma_16816<__half>(part[nt][0], a00, a10, a01, a11, qf[nt][2 * i][2 * k], qf[nt][2 * i][2 * k + 1]);
        mma_16816<__half>(part[nt][1], a02, a12, a03, a13, qf[nt][2 * i + 1][2 * k], qf[nt][2 * i + 1][2 * k + 1]);
      }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int k = 0; k < 4; ++k) sc[nt][k] = part[nt][0][k] + part[nt][1][k];
}
// V: code and scale places in the rows of the keys 2t (0) and 2t + 1 (1), dims g * D/8
// ..; bits of `gone`: keys 2t, 2t + 1, 2t + 8, 2t + 9 that count as zero.
template <int D, int NT, int QS>
__device__ __forceinline__ void pv_fp4(float (&o)[NT][D / 16][4], const float (&p)[NT][4], const uint8_t* code0,
                                       const uint8_t* code1, const uint8_t* scale0, const uint8_t* scale1, uint32_t gone) {
  uint32_t pb[NT][2 * QS];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    pb[nt][0] = movmatrix_trans(pack16<__half>(p[nt][0], p[nt][1]));
    pb[nt][1] = movmatrix_trans(pack16<__half>(p[nt][2], p[nt][3]));
    if constexpr (QS == 2) {
      auto rest = [](float x) { return x - __half2float(__float2half_rn(x)); };
      pb[nt][2] = movmatrix_trans(pack16<__half>(rest(p[nt][0]), rest(p[nt][1])));
      pb[nt][3] = movmatrix_trans(pack16<__half>(rest(p[nt][2]), rest(p[nt][3])));
    }
  }
  uint32_t c[4][D / 64], sb[4];
  const uint8_t* code[4] = {code0, code1, code0 + 8 * (D / 2), code1 + 8 * (D / 2)};
  const uint8_t* scale[4] = {scale0, scale1, scale0 + 8 * (D / 16), scale1 + 8 * (D / 16)};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (D == 128) {
      const uint2 v = *reinterpret_cast<const uint2*>(code[k]);
      c[k][0] = v.x;
      c[k][1] = v.y;
    } else {
      c[k][0] = *reinterpret_cast<const uint32_t*>(code[k]);
    }
    sb[k] = *scale[k];
  }
  if (gone) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (gone >> k & 1u) sb[k] = 0u;
  }
  const uint32_t s01 = e4m3x2_to_half2(sb[0] | (sb[1] << 8)), s23 = e4m3x2_to_half2(sb[2] | (sb[3] << 8));
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    // nibble pairs (key 2t, key 2t + 1) of the even and of the odd dims
    const uint32_t ev0 = (c[0][i] & 0x0F0F0F0Fu) | ((c[1][i] << 4) & 0xF0F0F0F0u);
    const uint32_t od0 = ((c[0][i] >> 4) & 0x0F0F0F0Fu) | (c[1][i] & 0xF0F0F0F0u);
    const uint32_t ev1 = (c[2][i] & 0x0F0F0F0Fu) | ((c[3][i] << 4) & 0xF0F0F0F0u);
    const uint32_t od1 = ((c[2][i] >> 4) & 0x0F0F0F0Fu) | (c[3][i] & 0xF0F0F0F0u);
    auto tile = [&](auto byte) {
      constexpr int B = decltype(byte)::value;
      const uint32_t f0 = mul_half2(e2m1x2_to_half2<B>(ev0), s01), f1 = mul_half2(e2m1x2_to_half2<B>(od0), s01);
      const uint32_t f2 = mul_half2(e2m1x2_to_half2<B>(ev1), s23), f3 = mul_half2(e2m1x2_to_half2<B>(od1), s23);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float(&acc)[4] = o[nt][4 * i + B];
        if constexpr (QS == 2) {
          float part[4] = {0.f, 0.f, 0.f, 0.f};
          mma_16816<__half>(part, f0, f1, f2, f3, pb[nt][2], pb[nt][3]);
          mma_16816<__half>(part, f0, f1, f2, f3, pb[nt][0], pb[nt][1]);
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[k] += part[k];
        } else {
          mma_16816<__half>(acc, f0, f1, f2, f3, pb[nt][0], pb[nt][1]);
        }
      }
    };
    tile(std::integral_constant<int, 0>{});
    tile(std::integral_constant<int, 1>{});
    tile(std::integral_constant<int, 2>{});
    tile(std::integral_constant<int, 3>{});
  }
}

template <typename T, typename KV, int D, int NT>
__global__ void __launch_bounds__(DecodeLayout<T, KV, D, NT>::kThreads, DecodeLayout<T, KV, D, NT>::kCtas)
    attn_paged_decode_kernel(const DecodeArgs d, const __grid_constant__ CUtensorMap tk,
                             const __grid_constant__ CUtensorMap tv) {
  using L = DecodeLayout<T, KV, D, NT>;
  using MT = typename std::conditional<L::kFp4, __half, T>::type;  // MMA operand type of 16-bit MMAs
  constexpr bool kF32 = L::kF32;
  constexpr int QS = L::kFp4 && std::is_same<T, float>::value ? 2 : 1;  // halves that make up a q or p
  constexpr int BN = L::BN, R = L::R, E = L::kEntries, W = L::W, SUB = L::SUB;
  extern __shared__ uint8_t smem_base[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_base) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* empty = full + E;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedAttnArgs& a = d.a;
  if (threadIdx.x == 0) {
    for (int s = 0; s < E; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], W);
    }
    mbar_fence_init();
  }
  if (threadIdx.x == 32 * W) {
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  Walker<BN, R> walk(d, lane);
  Segment seg;
  // 4-bit pages: a (page, head) block is copied as it is, codes then scales
  const int block_rows = 1 << a.seqs.page_shift, block_bytes = block_rows * D * 9 / 16;
  if (warp == W) {
    // ---- producer: page ids (32 at a time, the next 32 already asked for) and TMA boxes
    const int shift = a.seqs.page_shift, page_rows = 1 << shift;
    const int box_rows = min(page_rows, BN), boxes = BN / box_rows;
    int at = 0;  // ring entries filled: 2 per block, K then V
    bool alive = true;
    while (alive && walk.get(seg)) {
      const int32_t* ids = a.seqs.page_table + seg.b * a.seqs.max_pages;
      const int first_page = seg.w.key_lo >> shift, last_page = (seg.w.kv_len - 1) >> shift;  // others may be gone
      const int none = static_cast<int>(a.seqs.num_pages);  // outside the map: reads as zeros
      auto fetch = [&](int chunk) {
        const int i = chunk * 32 + lane;
        return i <= last_page ? ids[i] : none;
      };
      int chunk = ((seg.block * BN) >> shift) >> 5;
      int cur = fetch(chunk), nxt = fetch(chunk + 1);
      for (int j = 0; j < seg.blocks && alive; ++j) {
        const int key0 = (seg.block + j) * BN;
        const int first = key0 >> shift;
        if ((first >> 5) != chunk) {
          ++chunk;
          cur = nxt;
          nxt = fetch(chunk + 1);
        }
        int page = __shfl_sync(0xffffffffu, cur, (first + lane) & 31);
        if (first + lane < first_page || first + lane > last_page) page = none;
        else if (lane < boxes && (page < 0 || page >= none)) {
          set_device_error(a.seqs.err, kDevErrPageIndex);
          page = none;
        }
        const int row = key0 & (page_rows - 1);  // 0 unless a page holds several blocks
        const int box_at = lane * box_rows;
#pragma unroll 1
        for (int which = 0; which < 2; ++which, ++at) {
          const int e = at % E;
          const bool free_entry = mbar_wait(&empty[e], ((at / E) & 1) ^ 1);
          if (!__all_sync(0xffffffffu, free_entry)) {
            if (lane == 0) set_device_error(a.seqs.err, kDevErrAttentionTimeout);
            alive = false;
            break;
          }
          uint8_t* dst = smem + e * L::kEntry;
          if constexpr (L::kFp4) {
            const bool copy = lane < boxes && page != none;
            uint8_t* block = dst + lane * block_bytes;
            // a bad page, or one behind the window: zeros, ordered before the arrival below
            // (for the consumers) and before a later copy into the entry (another proxy)
            if (lane < boxes && page == none && first + lane <= last_page) {
              for (int i = 0; i < block_bytes; i += 16) *reinterpret_cast<uint4*>(block + i) = make_uint4(0u, 0u, 0u, 0u);
              fence_proxy_async_smem();
            }
            __syncwarp();
            const int copies = __popc(__ballot_sync(0xffffffffu, copy));
            if (lane == 0) mbar_arrive_expect_tx(&full[e], static_cast<uint32_t>(copies * block_bytes));
            __syncwarp();
            if (copy)
              bulk_load(block, static_cast<const uint8_t*>(which ? a.v_pages : a.k_pages) +
                                   (static_cast<int64_t>(page) * a.hkv + seg.kvh) * block_bytes,
                        static_cast<uint32_t>(block_bytes), &full[e]);
          } else {
            if (lane == 0) mbar_arrive_expect_tx(&full[e], L::kEntry);
            __syncwarp();
            if (lane < boxes) {
              const CUtensorMap* map = which ? &tv : &tk;
              constexpr int kBoxWidth = kF32 ? 128 : 64;  // in the map's units: bytes or 16-bit elements
#pragma unroll
              for (int c = 0; c < L::kRowBytes / 128; ++c)
                tma_load_4d(dst + c * L::kBox + box_at * 128, map, c * kBoxWidth, row, seg.kvh, page, &full[e]);
            }
          }
          __syncwarp();
        }
      }
    }
    // no copy may still be writing shared memory when the CTA exits
    for (int i = max(0, at - E); i < at; ++i) mbar_wait(&full[i % E], (i / E) & 1);
    return;
  }

  // ---- consumers
  const int g = lane >> 2, t = lane & 3;
  float* merge = reinterpret_cast<float*>(smem + L::kMergeOff);
  float* wm = reinterpret_cast<float*>(smem + L::kMlOff);  // [W][R]
  float* wl = wm + W * R;
  // MMA key row x of a 16-key group holds key perm(x): the fragment reads of 4-bit V
  // and of float32 K and V then fall into different banks
  // (4-bit at D 128: two of the four keys still share banks)
  auto perm = [](int x) {
    if (L::kFp4 && D == 128) return x ^ ((x >> 1) & 1);
    return L::kFp4 || kF32 ? (x & 8) | ((x & 6) >> 1) | ((x & 1) << 2) : x;
  };
  const float cap2 = 2.f * a.softcap * kLog2e;
  const float base_scale = a.softcap > 0.f ? a.scale * 2.f * kLog2e / a.softcap : a.scale * kLog2e;
  int at = 0;  // ring entries consumed
  bool alive = true;
  const int kw = warp * 16;  // this warp's keys of every block (and of each further 16 W)
  // 4-bit pages: places of the warp's 16-key groups in an entry, and this thread's in a group
  int code_off[SUB], scale_off[SUB];
#pragma unroll
  for (int u = 0; u < SUB; ++u) {
    const int r = kw + u * 16 * W, at_block = (r >> a.seqs.page_shift) * block_bytes;
    code_off[u] = at_block + (r & (block_rows - 1)) * (D / 2);
    scale_off[u] = at_block + block_rows * (D / 2) + (r & (block_rows - 1)) * (D / 16);
  }
  const int kcode = perm(g) * (D / 2) + t * (D / 8), kscale = perm(g) * (D / 16) + t * (D / 64);
  const int vcode0 = perm(2 * t) * (D / 2) + g * (D / 16), vcode1 = perm(2 * t + 1) * (D / 2) + g * (D / 16);
  const int vscale0 = perm(2 * t) * (D / 16) + g * (D / 8) / 16, vscale1 = perm(2 * t + 1) * (D / 16) + g * (D / 8) / 16;

  while (walk.get(seg)) {
    const int rows_left = seg.w.rows.n * a.group - seg.rt * R;
    const int rows = min(rows_left, R);
    // the two score columns of this thread in each n8 tile: rows nt * 8 + 2t + e
    int pos[NT][2];
    float slope[NT][2], rscale[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = nt * 8 + 2 * t + e;
        const int rr = seg.rt * R + min(r, rows - 1);
        const int tok = rr / a.group;
        pos[nt][e] = seg.w.rows.past + tok;
        slope[nt][e] = a.slopes ? a.slopes[seg.kvh * a.group + rr - tok * a.group] * kLog2e : 0.f;
        rscale[nt][e] = base_scale;
      }
    // Q^T fragments, rows past the tile zero
    constexpr int KK = D / 16;
    constexpr int QR = kF32 ? 4 : 2 * QS;  // registers per 16 dims
    uint32_t qf[NT][KK][QR];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + g;
      const bool valid = r < rows;
      const int rr = seg.rt * R + (valid ? r : 0);
      const int tok = rr / a.group, h = seg.kvh * a.group + rr - tok * a.group;
      const T* q = static_cast<const T*>(a.q) + ((seg.w.rows.row0 + tok) * a.hq + h) * D;
      if constexpr (L::kFp4) {
        // dims [t * D/4, (t + 1) * D/4) in order: the k order of the MMAs is that of the code bytes
        float x[D / 4];
        float big = 0.f;
#pragma unroll
        for (int v = 0; v < D / 4; v += Vec16<T>::N) {
          const Vec16<T> in = load16(q + t * (D / 4) + v);
#pragma unroll
          for (int j = 0; j < Vec16<T>::N; ++j) {
            x[v + j] = valid ? to_f32(in.e[j]) : 0.f;
            big = fmaxf(big, fabsf(x[v + j]));
          }
        }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        // 2^-e with 2^e <= max|q| < 2^(e+1), e within +-120
        const int e = max(-120, min(120, static_cast<int>((__float_as_uint(big) >> 23) & 255u) - 127));
        const float down = __uint_as_float(static_cast<unsigned>(127 - e) << 23);
        const float up = __uint_as_float(static_cast<unsigned>(127 + e) << 23);
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          const float u = x[2 * j] * down, w = x[2 * j + 1] * down;
          qf[nt][j / 2][j & 1] = pack16<__half>(u, w);
          if constexpr (QS == 2)
            qf[nt][j / 2][2 + (j & 1)] = pack16<__half>(u - __half2float(__float2half_rn(u)), w - __half2float(__float2half_rn(w)));
        }
        rscale[nt][0] *= __shfl_sync(0xffffffffu, up, (2 * t) * 4);
        rscale[nt][1] *= __shfl_sync(0xffffffffu, up, (2 * t + 1) * 4);
      } else if constexpr (kF32) {
        // MMA pair kk: dims kk * 16 + 4t .. + 3
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          const uint4 v = *reinterpret_cast<const uint4*>(q + kk * 16 + 4 * t);
          qf[nt][kk][0] = valid ? v.x : 0u;
          qf[nt][kk][1] = valid ? v.y : 0u;
          qf[nt][kk][2] = valid ? v.z : 0u;
          qf[nt][kk][3] = valid ? v.w : 0u;
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            qf[nt][kk][e] = valid ? *reinterpret_cast<const uint32_t*>(q + kk * 16 + e * 8 + 2 * t) : 0u;
      }
    }
    float o[NT][KK][4];
    float m[NT][2], l[NT][2], mul[NT][2];  // mul: what turns a masked score into log2 units
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // a scale that underflows (of a q of zeros over 4-bit pages, say) must not make NaN of
      // a masked score's -inf: no score is above 2^-100 with either
      mul[nt][0] = a.softcap > 0.f || a.slopes ? 1.f : fmaxf(rscale[nt][0], FLT_MIN);
      mul[nt][1] = a.softcap > 0.f || a.slopes ? 1.f : fmaxf(rscale[nt][1], FLT_MIN);
#pragma unroll
      for (int i = 0; i < KK; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }

    for (int j = 0; j < seg.blocks; ++j) {
      // waits for ring entry `at`; one that runs out skips the remaining blocks, with
      // every barrier of the CTA still met
      auto arrived = [&]() {
        const bool got = mbar_wait(&full[at % E], (at / E) & 1);
        if (!__all_sync(0xffffffffu, got)) {
          if (lane == 0) set_device_error(a.seqs.err, kDevErrAttentionTimeout);
          alive = false;
        }
        return alive;
      };
      auto release = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[at % E]);
        ++at;
      };
      if (!alive || !arrived()) continue;
      const uint8_t* sk = smem + (at % E) * L::kEntry;
      const int blk_key = (seg.block + j) * BN;

      float sc[SUB][NT][4];  // S^T: key rows g, g + 8 of the group, query rows 2t, 2t + 1
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        if constexpr (L::kFp4) qk_fp4<D, NT, QS>(sc[u], sk + code_off[u] + kcode, sk + scale_off[u] + kscale, qf);
        else if constexpr (kF32) qk_f32<D, NT>(sc[u], sk, L::kBox, kw + u * 16 * W, g, t, qf);
        else qk_16<T, D, NT>(sc[u], smem_u32(sk), L::kBox, kw + u * 16 * W, lane, qf);
      }
      release();

      // cap and bias (into log2 units), mask
      if (a.softcap > 0.f || a.slopes) {
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float x = sc[u][nt][i] * rscale[nt][i & 1];
              if (a.softcap > 0.f) x = capped_score(x, cap2);
              const int key = blk_key + u * 16 * W + kw + perm(g + (i >> 1) * 8);
              sc[u][nt][i] = fmaf(slope[nt][i & 1], static_cast<float>(key - pos[nt][i & 1]), x);
            }
      }
      if (blk_key + BN > seg.w.rows.past + 1 || blk_key < seg.w.kv_len - a.window) {
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = blk_key + u * 16 * W + kw + perm(g + (i >> 1) * 8), at_pos = pos[nt][i & 1];
              if (key > at_pos || key <= at_pos - a.window) sc[u][nt][i] = -INFINITY;
            }
      }
      // running maximum; O and the sums are rescaled when it moves
      float top[NT][2];
      bool moved = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(sc[0][nt][e], sc[0][nt][e + 2]);
#pragma unroll
          for (int u = 1; u < SUB; ++u) x = fmaxf(x, fmaxf(sc[u][nt][e], sc[u][nt][e + 2]));
#pragma unroll
          for (int s = 4; s < 32; s <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, s));
          top[nt][e] = fmaxf(m[nt][e], x * mul[nt][e]);
          moved |= top[nt][e] != m[nt][e];
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float alpha[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            alpha[e] = m[nt][e] == top[nt][e] ? 1.f : exp2_approx(m[nt][e] - top[nt][e]);  // from -inf: 0
            m[nt][e] = top[nt][e];
            l[nt][e] *= alpha[e];
          }
#pragma unroll
          for (int i = 0; i < KK; ++i) {
            o[nt][i][0] *= alpha[0];
            o[nt][i][1] *= alpha[1];
            o[nt][i][2] *= alpha[0];
            o[nt][i][3] *= alpha[1];
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // a row that has seen no key yet keeps m = -inf: its p are 0
          const float neg = m[nt][e] == -INFINITY ? 0.f : -m[nt][e];
#pragma unroll
          for (int u = 0; u < SUB; ++u) {
            sc[u][nt][e] = exp2_approx(fmaf(sc[u][nt][e], mul[nt][e], neg));
            sc[u][nt][e + 2] = exp2_approx(fmaf(sc[u][nt][e + 2], mul[nt][e], neg));
            l[nt][e] += sc[u][nt][e] + sc[u][nt][e + 2];  // this thread's keys; summed over the warp at the end
          }
        }

      // O^T += V^T P^T
      if (!arrived()) continue;
      uint8_t* sv = smem + (at % E) * L::kEntry;
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        const int key_first = blk_key + u * 16 * W + kw;
        // rows that are not of the sequence may hold anything: a zero weight must meet a zero
        const bool stale = key_first + 16 > seg.w.kv_len || key_first < seg.w.key_lo;
        auto foreign = [&](int r) { return key_first + r >= seg.w.kv_len || key_first + r < seg.w.key_lo; };
        if constexpr (L::kFp4) {
          uint32_t gone = 0u;  // of the keys 2t, 2t + 1, 2t + 8, 2t + 9
          if (stale) {
#pragma unroll
            for (int k = 0; k < 4; ++k) gone |= static_cast<uint32_t>(foreign(perm(2 * t + (k & 1) + (k >> 1) * 8))) << k;
          }
          pv_fp4<D, NT, QS>(o, sc[u], sv + code_off[u] + vcode0, sv + code_off[u] + vcode1, sv + scale_off[u] + vscale0,
                            sv + scale_off[u] + vscale1, gone);
        } else {
          if (stale) {
            for (int c = lane; c < 16 * (L::kRowBytes / 16); c += 32) {
              const int r = (c >> 3) & 15, box = c >> 7;
              if (foreign(r))
                *reinterpret_cast<uint4*>(sv + box * L::kBox + (kw + u * 16 * W + r) * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();  // before the entry is given back to the TMA
            __syncwarp();
          }
          if constexpr (kF32) pv_f32<D, NT>(o, sc[u], sv, L::kBox, kw + u * 16 * W, g, t);
          else pv_16<T, D, NT>(o, sc[u], smem_u32(sv), L::kBox, kw + u * 16 * W, lane);
        }
      }
      release();
    }

    // ---- merge the warps in order, then store the rows or the part
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], s);
        if (g == 0) {
          wm[warp * R + nt * 8 + 2 * t + e] = m[nt][e];
          wl[warp * R + nt * 8 + 2 * t + e] = l[nt][e];
        }
      }
    asm volatile("bar.sync 1, %0;" ::"n"(32 * W) : "memory");
    constexpr int DH = L::DH;
#pragma unroll
    for (int half = 0; half < D / DH; ++half) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nt * 8 + 2 * t + e;
          float top = -INFINITY;
#pragma unroll
          for (int w = 0; w < W; ++w) top = fmaxf(top, wm[w * R + r]);
          f[e] = m[nt][e] == -INFINITY ? 0.f : exp2_approx(m[nt][e] - top);
        }
#pragma unroll
        for (int i = 0; i < KK; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            // 16-bit: dims i * 16 + g (+ 8); 4-bit: g * D/8 + 2 i (+ 1); float32: see the reads of V
            const int dim = L::kFp4 ? g * (D / 8) + 2 * i + (k >> 1)
                            : kF32  ? 32 * (i >> 1) + 4 * f32_chunk(g) + 2 * (i & 1) + (k >> 1)
                                    : i * 16 + g + (k >> 1) * 8;
            if (D == DH || dim / DH == half)
              merge[(warp * R + nt * 8 + 2 * t + (k & 1)) * DH + (dim - half * DH)] = o[nt][i][k] * f[k & 1];
          }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(32 * W) : "memory");
      for (int c = threadIdx.x; c < rows * (DH / 4); c += 32 * W) {
        const int r = c / (DH / 4), x = (c - r * (DH / 4)) * 4;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        float top = -INFINITY, den = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, wm[w * R + r]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float4 v = *reinterpret_cast<const float4*>(&merge[(w * R + r) * DH + x]);
          sum.x += v.x;
          sum.y += v.y;
          sum.z += v.z;
          sum.w += v.w;
          const float mw = wm[w * R + r];
          // without a score above -inf the sum is 0, or NaN
          den += mw == -INFINITY ? wl[w * R + r] : wl[w * R + r] * exp2_approx(mw - top);
        }
        const int dim = half * DH + x;
        if (seg.whole) {
          const int rr = seg.rt * R + r, tok = rr / a.group, h = seg.kvh * a.group + rr - tok * a.group;
          const float inv = a.v_scale / den;
          store4(static_cast<T*>(a.out) + ((seg.w.rows.row0 + tok) * a.hq + h) * D + dim, sum.x * inv, sum.y * inv,
                 sum.z * inv, sum.w * inv);
        } else {
          *reinterpret_cast<float4*>(d.part_o + (static_cast<int64_t>(seg.slot) * R + r) * D + dim) = sum;
          if (dim == 0) d.part_ml[static_cast<int64_t>(seg.slot) * R + r] = make_float2(top, den);
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(32 * W) : "memory");
    }
  }
}

// Merges the parts of the units that were split, in the order of the list: the first
// part's slot is its CTA's first or second, the others are the first slots of the
// CTAs after it. grid = (units, D / 32); thread = (parts lane, row, 4 dims). Which
// parts there are is worked out while the main kernel still runs: positions and starts
// were final before that began.
template <typename T, int D, int BN, int R>
__global__ void __launch_bounds__(256) attn_paged_combine_kernel(const DecodeArgs d) {
  const PagedAttnArgs& a = d.a;
  const int u = blockIdx.x, rt = u % d.tiles_max, kvh = u / d.tiles_max % a.hkv, b = u / d.tiles_max / a.hkv;
  const int lane = threadIdx.x & 31;
  constexpr int ITEMS = R * 8, LANES = 256 / ITEMS;
  __shared__ float4 so[LANES][ITEMS];
  __shared__ float2 sml[LANES][ITEMS];

  const SeqWork sw = seq_work<BN, R>(a, b, false);
  const int rows = min(sw.rows.n * a.group - rt * R, R);
  int total = 0, base = 0;
  for (int c = 0; c < a.seqs.batch; c += 32) {
    if (c + lane < a.seqs.batch) {
      const SeqWork s = seq_work<BN, R>(a, c + lane, false);
      const int work = a.hkv * s.tiles * s.blocks;
      total += work;
      if (c + lane < b) base += work;
    }
  }
  total = __reduce_add_sync(0xffffffffu, total);
  base = __reduce_add_sync(0xffffffffu, base);
  const Shares shares(total, d.ctas, d.min_blocks);
  const int begin = base + (kvh * sw.tiles + rt) * sw.blocks;
  int first = 0, parts = 1;
  if (rows > 0) {
    first = shares.cta_of(begin);
    parts = shares.cta_of(begin + sw.blocks - 1) - first + 1;
  }
  pdl_wait();
  pdl_trigger();
  if (rows <= 0 || parts == 1) return;  // uniform for the CTA

  const int item = threadIdx.x % ITEMS, pl = threadIdx.x / ITEMS;
  const int r = item >> 3, dim = blockIdx.y * 32 + (item & 7) * 4;
  const int slot0 = begin == shares.begin(first) ? 2 * first : 2 * first + 1;
  float top = -INFINITY, den = 0.f;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  if (r < rows) {
    for (int p0 = pl; p0 < parts; p0 += 4 * LANES) {
      float2 ml[4];
      float4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int p = p0 + k * LANES;
        ml[k] = make_float2(-INFINITY, 0.f);
        v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p < parts) {
          const int64_t slot = p == 0 ? slot0 : 2 * (first + p);
          ml[k] = d.part_ml[slot * R + r];
          v[k] = *reinterpret_cast<const float4*>(d.part_o + (slot * R + r) * D + dim);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // a part in which the row sees no key (the sum of one whose scores are all NaN is NaN)
        if (ml[k].x == -INFINITY && ml[k].y == 0.f) continue;
        const float m = fmaxf(top, ml[k].x);
        const float f = exp2_approx(top - m), f2 = exp2_approx(ml[k].x - m);  // top = -inf: 0
        top = m;
        den = den * f + ml[k].y * f2;
        sum.x = sum.x * f + v[k].x * f2;
        sum.y = sum.y * f + v[k].y * f2;
        sum.z = sum.z * f + v[k].z * f2;
        sum.w = sum.w * f + v[k].w * f2;
      }
    }
  }
  so[pl][item] = sum;
  sml[pl][item] = make_float2(top, den);
  __syncthreads();
  if (pl > 0 || r >= rows) return;
#pragma unroll
  for (int k = 1; k < LANES; ++k) top = fmaxf(top, sml[k][item].x);
  den = 0.f;
  sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int k = 0; k < LANES; ++k) {
    const float2 ml = sml[k][item];
    const float4 v = so[k][item];
    const float f = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - top);
    den += ml.y * f;
    sum.x += v.x * f;
    sum.y += v.y * f;
    sum.z += v.z * f;
    sum.w += v.w * f;
  }
  const int rr = rt * R + r, tok = rr / a.group, h = kvh * a.group + rr - tok * a.group;
  const float inv = a.v_scale / den;
  store4(static_cast<T*>(a.out) + ((sw.rows.row0 + tok) * a.hq + h) * D + dim, sum.x * inv, sum.y * inv, sum.z * inv,
         sum.w * inv);
}

// ---- host ------------------------------------------------------------------------

// CTAs that are resident at once, per kernel and device.
int resident_ctas(const void* kernel, int threads, int smem) {
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, int> cache;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  std::lock_guard<std::mutex> lock(mu);
  auto it = cache.find({dev, kernel});
  if (it != cache.end()) return it->second;
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess) {
    cudaGetLastError();
    n = 0;
  }
  n *= sm_count();
  cache[{dev, kernel}] = n;
  return n;
}

struct DecodePlan {
  int nt, tiles_max;
  bool split;
  int64_t units, grid;
  size_t part_o, part_ml, workspace;
};

// Shares of a split call are at least kMinKeys keys (1 x 1501 keys, us with 64 | 128 |
// 256 | 512: 28/4 heads 16 bits 8.3 | 8.4 | 9.9 | 13.5, 4 bits 8.5 | 8.5 | 9.6 | 11.9,
// float32 16/4 heads 10.5 | 11.6 | 15.1 | 23.3; nothing changes where every CTA has
// more); a call whose sequences cannot exceed kWholeKeys runs one CTA per unit.
constexpr int kWholeKeys = 512;
constexpr int kMinKeys = 128;
constexpr int kMaxCtasPerSm = 3;

// max_keys: that a row may see; table_keys: the table's rows. The size of the workspace is
// asked for without a window (max_keys = table_keys), so whatever calls for one goes by
// the table, and a window can only take the need away.
DecodePlan plan_paged_decode(int64_t batch, int64_t hkv, int64_t group, int64_t max_new, int64_t head_dim, int64_t max_keys,
                             int64_t table_keys, bool f32) {
  DecodePlan p{};
  const int64_t rows = group * max_new;
  p.nt = rows <= 8 || f32 ? 1 : 2;  // two row tiles of split operands do not fit the registers
  p.tiles_max = static_cast<int>(ceil_div(rows, 8 * p.nt));
  p.units = batch * hkv * p.tiles_max;
  // the list's length has to fit an int (a longer one is never short of CTAs)
  p.split = max_keys > kWholeKeys && p.units * (table_keys / 64 + 2) < INT_MAX;
  p.grid = p.split ? static_cast<int64_t>(sm_count()) * kMaxCtasPerSm : p.units;
  if (p.split) {
    const int64_t r = 8 * p.nt;
    p.part_o = static_cast<size_t>(2 * p.grid * r * head_dim) * 4;
    p.part_ml = static_cast<size_t>(2 * p.grid * r) * 8;
    p.workspace = p.part_o + p.part_ml;
  }
  return p;
}

template <typename T, typename KV, int D, int NT>
dli_status launch_paged_decode(const PagedAttnArgs& a, const DecodePlan& plan, void* workspace, cudaStream_t stream) {
  using L = DecodeLayout<T, KV, D, NT>;
  CUtensorMap tk{}, tv{};  // not used for 4-bit pages
  const int64_t page_rows = 1ll << a.seqs.page_shift;
  const dli_dtype kv_dtype = L::kF32                                 ? DLI_DTYPE_F32
                             : std::is_same<T, __nv_bfloat16>::value ? DLI_DTYPE_BF16
                                                                       : DLI_DTYPE_F16;
  dli_status st = L::kFp4 ? DLI_OK : make_page_maps(a, kv_dtype, D, static_cast<int>(std::min<int64_t>(page_rows, L::BN)), &tk, &tv);
  if (st != DLI_OK) return st;
  auto kern = attn_paged_decode_kernel<T, KV, D, NT>;
  st = ensure_smem(reinterpret_cast<const void*>(kern), L::kBytes, "attention_paged");
  if (st != DLI_OK) return st;
  DecodeArgs d{};
  d.a = a;
  d.tiles_max = plan.tiles_max;
  d.split = plan.split ? 1 : 0;
  d.min_blocks = std::max(1, kMinKeys / L::BN);
  int64_t grid = plan.grid;
  if (plan.split) {
    d.part_o = static_cast<float*>(workspace);
    d.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + plan.part_o);
    grid = std::min<int64_t>(grid, std::max(1, resident_ctas(reinterpret_cast<const void*>(kern), L::kThreads, L::kBytes)));
    d.ctas = static_cast<int>(grid);
  }
  launch_pdl(kern, dim3(static_cast<unsigned>(grid)), dim3(L::kThreads), L::kBytes, stream, d, tk, tv);
  if (plan.split)
    launch_pdl(attn_paged_combine_kernel<T, D, L::BN, L::R>, dim3(static_cast<unsigned>(plan.units), D / 32), dim3(256), 0, stream, d);
  return check_launch("attention_paged", plan.split ? 2 : 1);
}

template <typename T, typename KV>
dli_status launch_paged_decode_nd(const PagedAttnArgs& a, const DecodePlan& plan, void* ws, cudaStream_t stream) {
  if constexpr (!std::is_same<T, float>::value)
    if (plan.nt == 2)
      return a.head_dim == 64 ? launch_paged_decode<T, KV, 64, 2>(a, plan, ws, stream) : launch_paged_decode<T, KV, 128, 2>(a, plan, ws, stream);
  return a.head_dim == 64 ? launch_paged_decode<T, KV, 64, 1>(a, plan, ws, stream) : launch_paged_decode<T, KV, 128, 1>(a, plan, ws, stream);
}

DecodePlan plan_of(const PagedAttnArgs& a, dli_dtype dtype) {
  const int64_t table_keys = a.seqs.max_pages << a.seqs.page_shift;
  return plan_paged_decode(a.seqs.batch, a.hkv, a.group, a.seqs.max_new, a.head_dim,
                           std::min<int64_t>(table_keys, static_cast<int64_t>(a.window) + a.seqs.max_new), table_keys,
                           dtype == DLI_DTYPE_F32);
}

}  // namespace

// 4-D maps over the pages: [num_pages, Hkv, page rows, D] 16-bit elements, or bytes of
// float32 elements.
dli_status make_page_maps(const PagedAttnArgs& a, dli_dtype dtype, int d, int box_rows, CUtensorMap* tk, CUtensorMap* tv) {
  const uint64_t page_rows = 1ull << a.seqs.page_shift, hkv = static_cast<uint64_t>(a.hkv);
  const uint64_t pages = static_cast<uint64_t>(a.seqs.num_pages), ud = static_cast<uint64_t>(d);
  const uint32_t rows = static_cast<uint32_t>(box_rows);
  const void* base[2] = {a.k_pages, a.v_pages};
  CUtensorMap* map[2] = {tk, tv};
  const uint64_t es = dtype_bytes(dtype);
  const uint64_t strides[3] = {ud * es, page_rows * ud * es, hkv * page_rows * ud * es};
  for (int i = 0; i < 2; ++i) {
    dli_status st;
    if (dtype == DLI_DTYPE_F32) {
      const uint64_t dims[4] = {ud * 4, page_rows, hkv, pages};
      const uint32_t box[4] = {128u, rows, 1u, 1u};
      st = make_map_4d_bytes(map[i], base[i], dims, strides, box);
    } else {
      const uint64_t dims[4] = {ud, page_rows, hkv, pages};
      const uint32_t box[4] = {64u, rows, 1u, 1u};
      st = make_map_4d(map[i], base[i], dtype == DLI_DTYPE_BF16, dims, strides, box);
    }
    if (st != DLI_OK) return st;
  }
  return DLI_OK;
}

bool paged_decode_serves(const PagedAttnArgs& a, dli_dtype dtype) {
  if (!is_float_dtype(dtype) || (a.head_dim != 64 && a.head_dim != 128)) return false;
  if (a.seqs.num_pages < 1) return false;
  for (const void* p : {a.q, a.k_pages, a.v_pages, static_cast<const void*>(a.out)})
    if (!aligned(p, 16)) return false;
  return plan_of(a, dtype).units <= INT_MAX;
}

size_t paged_decode_workspace(int64_t batch, int64_t hkv, int64_t group, int64_t max_new, int64_t head_dim, int64_t max_keys,
                              dli_dtype dtype) {
  return plan_paged_decode(batch, hkv, group, max_new, head_dim, max_keys, max_keys, dtype == DLI_DTYPE_F32).workspace;
}

dli_status run_paged_decode(const PagedAttnArgs& a, dli_dtype dtype, dli_dtype kv_dtype, void* workspace,
                            size_t workspace_bytes, cudaStream_t stream) {
  const DecodePlan plan = plan_of(a, dtype);
  if (plan.workspace > 0 && (workspace == nullptr || workspace_bytes < plan.workspace || !aligned(workspace, 16)))
    return fail(DLI_ERR_WORKSPACE, "attention_paged: a 16-byte aligned workspace of " + std::to_string(plan.workspace) + " bytes is needed");
  const bool fp4 = kv_dtype == DLI_DTYPE_FP4;
  if (dtype == DLI_DTYPE_F32)
    return fp4 ? launch_paged_decode_nd<float, Fp4>(a, plan, workspace, stream)
               : launch_paged_decode_nd<float, float>(a, plan, workspace, stream);
  if (dtype == DLI_DTYPE_BF16)
    return fp4 ? launch_paged_decode_nd<__nv_bfloat16, Fp4>(a, plan, workspace, stream)
               : launch_paged_decode_nd<__nv_bfloat16, __nv_bfloat16>(a, plan, workspace, stream);
  return fp4 ? launch_paged_decode_nd<__half, Fp4>(a, plan, workspace, stream)
             : launch_paged_decode_nd<__half, __half>(a, plan, workspace, stream);
}

}  // namespace dli_sm100
