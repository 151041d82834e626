// Paged KV cache: the append with rotary embedding, the gather of cached rows,
// and the entry points of the attention over pages with its general kernel.
//
// Pages are [num_pages, Hkv, page_size, D] of the model's type, or 4-bit: per
// (page, head) the rows' E2M1 codes, then their E4M3 scales, one per 16 elements.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "mma_sync.cuh"
#include "paged_attn.cuh"

namespace dli_sm100 {
namespace {

// ---- 4-bit blocks ------------------------------------------------------------------

// The float nearest to x toward zero, its last bit set when x is not that float:
// comparisons with any float of fewer than 24 bits come out as they do for x.
__device__ __forceinline__ float round_to_odd(double x) {
  const float f = __double2float_rz(x);
  return static_cast<double>(f) == x ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

// E4M3 code nearest to most / 6 (ties to the even code, at most 448). `most` is
// rounded to odd, and six times the midpoint of two neighbouring codes has at
// most 7 bits, so the comparison decides as the exact value would.
__device__ __forceinline__ unsigned e4m3_scale(float most) {
  const float t = most * (1.f / 6.f);
  const unsigned c = __nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3);
  const float v = e4m3_value(c);
  const unsigned up = t > v ? 1u : 0u;  // which neighbour could be nearer
  if (up ? c >= 126u : c == 0u) return c;
  const float mid = 3.f * (v + e4m3_value(up ? c + 1u : c - 1u));
  const bool odd_tie = most == mid && (c & 1u);
  if (up ? most > mid || odd_tie : most < mid || odd_tie) return up ? c + 1u : c - 1u;
  return c;
}

// The code word of 8 values (rounded to odd where they are not exact) for scale value
// s > 0, from its definition: a value's code is the number of rounding borders at or
// below it: 0.25, 0.75, ... times the scale, products of 3-bit numbers, hence exact; a
// border itself goes to the even code, so those below an even code count from the next
// float on.
__device__ __forceinline__ unsigned fp4_codes_by_borders(const float (&x)[8], float s) {
  auto after = [](float v) { return __uint_as_float(__float_as_uint(v) + 1u); };
  const float b0 = after(0.25f * s), b1 = 0.75f * s, b2 = after(1.25f * s), b3 = 1.75f * s, b4 = after(2.5f * s),
              b5 = 3.5f * s, b6 = after(5.f * s);
  unsigned w = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(x[i]);
    const bool hi = a >= b3, mid = a >= (hi ? b5 : b1);
    const bool low = a >= (hi ? (mid ? b6 : b4) : (mid ? b2 : b0));
    const unsigned c = (hi ? 4u : 0u) | (mid ? 2u : 0u) | (low ? 1u : 0u) | (x[i] < 0.f ? 8u : 0u);
    w |= c << (4 * i);
  }
  return w;
}
// The same by division and the conversion instruction: q = x / s correctly rounded
// (one Newton step from the rounded reciprocal), so a quotient that is a border comes
// out as it, and the conversion rounds ties to even. Only a q that is a border while
// x / s is not could go wrong; such a word is left to the comparisons.
__device__ __forceinline__ unsigned fp4_codes(const float (&x)[8], float s) {
  const float inv = __frcp_rn(s), most = 7.f * s;  // 6 s is the largest value: further out only saturates
  float q[8];
  bool doubt = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = fminf(fmaxf(x[i], -most), most);
    const float q0 = v * inv;
    q[i] = fmaf(fmaf(-q0, s, v), inv, q0);
    doubt |= (__float_as_uint(q[i]) & 0x000FFFFFu) == 0u && fmaf(-q[i], s, v) != 0.f;
  }
  if (doubt) return fp4_codes_by_borders(x, s);
  unsigned w = 0u;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    unsigned byte;  // + 0: a code for -0 has no sign
    asm("{.reg .b8 b; cvt.rn.satfinite.e2m1x2.f32 b, %1, %2; cvt.u32.u8 %0, b;}" : "=r"(byte) : "f"(q[i + 1] + 0.f), "f"(q[i] + 0.f));
    w |= byte << (4 * i);
  }
  return w;
}

// ---- append ------------------------------------------------------------------------
// The heads [head0, head1) of a token on per_pass x (D / V) threads, `tokens` tokens to
// a CTA.
struct HeadSplit {
  int head0, head1, per_pass, passes, tokens;
};

struct AppendArgs {
  PagedSeqs seqs;
  const void* qkv;
  const float* cos_t;
  const float* sin_t;
  void* q_out;
  void* k_pages;
  void* v_pages;
  int hq, hkv, head_dim, pairs;
  int64_t table_rows;
  float k_scale, v_scale;
  HeadSplit all, q, kv;
  int vec_tables;  // cos/sin rows can be read by 16 bytes
};

// V elements of T as they lie in memory: 16-byte vectors where they fill any.
template <typename T, int V>
struct Row {
  static constexpr int kVecs = V * static_cast<int>(sizeof(T)) / 16;
  union {
    uint4 raw[kVecs > 0 ? kVecs : 1];
    uint32_t w[V * sizeof(T) >= 4 ? V * sizeof(T) / 4 : 1];
    T e[V];
  };
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kVecs > 0) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) raw[i] = *reinterpret_cast<const uint4*>(p + i * Vec16<T>::N);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kVecs > 0) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) *reinterpret_cast<uint4*>(p + i * Vec16<T>::N) = raw[i];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = e[i];
    }
  }
  __device__ __forceinline__ float2 pair(int j) const {
    if constexpr (std::is_same<T, float>::value) return make_float2(e[2 * j], e[2 * j + 1]);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
      return make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
  }
  __device__ __forceinline__ void set_pair(int j, float x, float y) {
    if constexpr (std::is_same<T, float>::value) {
      e[2 * j] = x;
      e[2 * j + 1] = y;
    } else {
      w[j] = pack16<T>(x, y);
    }
  }
};

// The append: out (x, y) = (x c - y s, x s + y c) for the pairs of q and k, v as it is.
// Bound by memory (every byte of q|k|v is read once and written once, the rotary row is
// read once per token and pass), and for a decode step by the latency of one chain of
// loads. A thread owns elements [vi * V, vi * V + V) of a token's head and takes NP heads a
// step, hl, hl + per_pass, ..., whose loads are asked for together; a CTA holds as many
// tokens as it has room for: 24 ragged prompts of up to 2048 tokens, 14/2 heads of 64, 157 MB
// in 29.5 us = 5.3 TB/s (three heads a step 31 us, one 45); a step of 32 sequences, 28/4 heads of 128,
// 2.3 us in a graph of launches (a CTA for every sequence and token up to max_new: 128
// sequences of one token 2.7 us, with a max_new of 128 57). Into 4-bit pages k and v are
// quantised from 64 bits, k through doubles (exact products of two floats, their sum
// rounded once) and a division per value: 16 ragged prompts of up to 2048 tokens, 28/4
// heads of 128, 99 us (180 with one kind of CTA and comparisons for codes); with cache
// scales other than 1, which divide every k and v in doubles, a quarter more (93 -> 116 us
// at another draw of lengths).
template <typename T, typename KV, int V, int NP>
__device__ __forceinline__ void append_rows(const AppendArgs& a, const HeadSplit& hs, int walker, int walkers, int part,
                                            int parts) {
  constexpr bool kFp4 = std::is_same<KV, Fp4>::value;
  constexpr int H = V / 2;  // pairs of a thread
  const int b = blockIdx.y;
  const int d = a.head_dim, ipr = d / V, heads = a.hq + 2 * a.hkv;
  const int per_token = hs.per_pass * ipr;
  const int tl = threadIdx.x / per_token, lane = threadIdx.x - tl * per_token;
  if (tl >= hs.tokens) return;
  const int hl = lane / ipr, vi = lane - hl * ipr;
  const SeqRows sr = seq_rows(a.seqs, b, true);
  const int page_rows = 1 << a.seqs.page_shift;
  const int first_pair = vi * H;
  const int turned = max(0, min(H, a.pairs - first_pair));  // pairs of this thread that rotate
  const bool full = 2 * a.pairs == d;
  const int32_t* ids = a.seqs.page_table + b * a.seqs.max_pages;
  const int head_step = hs.per_pass * d;
  const int page_bytes = a.hkv * (page_rows * d * 9 / 16);  // of 4-bit pages
  for (int t = walker * hs.tokens + tl; t < sr.n; t += walkers * hs.tokens) {
    const int p = sr.past + t;
    const int64_t row = sr.row0 + t;
    for (int pass = part * NP; pass < hs.passes; pass += parts * NP) {
      // everything the rows need is asked for before any of it is looked at
      const int h0 = hs.head0 + hl + pass * hs.per_pass;
      const T* src = static_cast<const T*>(a.qkv) + row * (heads * d) + h0 * d + vi * V;
      T* q_row = static_cast<T*>(a.q_out) + row * (a.hq * d) + vi * V;
      Row<T, V> x[NP];
#pragma unroll
      for (int k = 0; k < NP; ++k)
        if (h0 + k * hs.per_pass < hs.head1) x[k].load(src + k * head_step);
      float c[H], s[H];
      const bool turn = turned > 0 && p < a.table_rows && h0 < a.hq + a.hkv;
      if (turn) {
        const float* ct = a.cos_t + static_cast<int64_t>(p) * a.pairs + first_pair;
        const float* st = a.sin_t + static_cast<int64_t>(p) * a.pairs + first_pair;
        if (H >= 4 && a.vec_tables) {
#pragma unroll
          for (int j = 0; j + 4 <= H; j += 4) {
            if (full || j < turned) {
              const float4 cv = *reinterpret_cast<const float4*>(ct + j), sv = *reinterpret_cast<const float4*>(st + j);
              c[j] = cv.x, c[j + 1] = cv.y, c[j + 2] = cv.z, c[j + 3] = cv.w;
              s[j] = sv.x, s[j + 1] = sv.y, s[j + 2] = sv.z, s[j + 3] = sv.w;
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < H; ++j) {
            if (j < turned) {
              c[j] = ct[j];
              s[j] = st[j];
            }
          }
        }
      } else if (turned > 0 && h0 < a.hq + a.hkv) {
        set_device_error(a.seqs.err, kDevErrRotaryPosition);
      }
      const int page = ids[p >> a.seqs.page_shift];
      const bool good = page >= 0 && page < a.seqs.num_pages;
      if (!good) set_device_error(a.seqs.err, kDevErrPageIndex);
      const int r = p & (page_rows - 1);
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const int h = h0 + k * hs.per_pass;
        if (h >= hs.head1) break;
        const bool is_q = h < a.hq, is_k = !is_q && h < a.hq + a.hkv;
        if (!is_q && !good) break;
        const int kvh = is_k ? h - a.hq : h - a.hq - a.hkv;
        if constexpr (kFp4) {
          if (!is_q) {
            static_assert(V == 8, "two threads share a block of 16");
            float f[V];
#pragma unroll
            for (int j = 0; j < H; ++j) {
              const float2 v = x[k].pair(j);
              f[2 * j] = v.x;
              f[2 * j + 1] = v.y;
            }
            const float cache_scale = is_k ? a.k_scale : a.v_scale;
            if (is_k || cache_scale != 1.f) {
              // products of a 24-bit and an at most 24-bit number are exact in 53 bits
#pragma unroll
              for (int j = 0; j < H; ++j) {
                double u = f[2 * j], w = f[2 * j + 1];
                if (is_k && turn && (full || j < turned)) {
                  const double cd = c[j], sd = s[j];
                  const double u0 = u * cd - w * sd;
                  w = u * sd + w * cd;
                  u = u0;
                }
                if (cache_scale != 1.f) {
                  u /= static_cast<double>(cache_scale);
                  w /= static_cast<double>(cache_scale);
                }
                f[2 * j] = round_to_odd(u);
                f[2 * j + 1] = round_to_odd(w);
              }
            }
            // the largest magnitude of the block, whose other half is the lane next door
            // (same token and head, so it is here too); as bits, a NaN is larger than any
            unsigned most = 0u;
#pragma unroll
            for (int j = 0; j < V; ++j) most = max(most, __float_as_uint(f[j]) & 0x7FFFFFFFu);
            most = max(most, __shfl_xor_sync(3u << (threadIdx.x & 30u), most, 1));
            const bool nan = most > 0x7F800000u;
            const unsigned scale = nan ? 0x7Fu : e4m3_scale(__uint_as_float(most));
            const float sv = nan ? 0.f : e4m3_value(scale);
            uint8_t* base = static_cast<uint8_t*>(is_k ? a.k_pages : a.v_pages) + static_cast<int64_t>(page) * page_bytes +
                            kvh * (page_rows * d * 9 / 16);
            *reinterpret_cast<unsigned*>(base + r * (d / 2) + vi * 4) = sv > 0.f ? fp4_codes(f, sv) : 0u;
            if ((vi & 1) == 0) base[page_rows * (d / 2) + r * (d / 16) + vi / 2] = static_cast<uint8_t>(scale);
            continue;
          }
        }
        if ((is_q || is_k) && turn) {
#pragma unroll
          for (int j = 0; j < H; ++j) {
            if (full || j < turned) {
              const float2 v = x[k].pair(j);
              x[k].set_pair(j, v.x * c[j] - v.y * s[j], v.x * s[j] + v.y * c[j]);
            }
          }
        }
        if (is_q) {
          x[k].store(q_row + h * d);
        } else {
          T* page_at = static_cast<T*>(is_k ? a.k_pages : a.v_pages) + static_cast<int64_t>(page) * (a.hkv * page_rows * d);
          x[k].store(page_at + (kvh * page_rows + r) * d + vi * V);
        }
      }
    }
  }
}

// grid = (token walkers, sequences, parts of the head passes).
template <typename T, typename KV, int V, int NP>
__global__ void __launch_bounds__(256, NP == 1 ? 2 : 4) qkv_rotary_paged_kernel(const AppendArgs a) {
  DLI_PDL_ENTRY();
  append_rows<T, KV, V, NP>(a, a.all, blockIdx.x, gridDim.x, blockIdx.z, gridDim.z);
}

// Many tokens into 4-bit pages: every other CTA streams q, four heads a thread, while its
// neighbours quantise k and v, two rows a thread (16 prompts, q heads | rows of k and v:
// 3 | 1 121 us, 3 | 2 113, 4 | 2 99, 3 | 4 120, 2 | 2 114), whose arithmetic then hides
// under the streaming. grid = (2 x token walkers, sequences).
template <typename T>
__global__ void __launch_bounds__(256, 4) qkv_rotary_paged_fp4_kernel(const AppendArgs a) {
  DLI_PDL_ENTRY();
  const int walker = blockIdx.x >> 1, walkers = gridDim.x >> 1;
  if (blockIdx.x & 1) append_rows<T, Fp4, 8, 2>(a, a.kv, walker, walkers, 0, 1);
  else append_rows<T, T, 8, 4>(a, a.q, walker, walkers, 0, 1);
}

template <typename T, typename KV, int V>
void launch_append(AppendArgs a, cudaStream_t stream) {
  constexpr bool kFp4 = std::is_same<KV, Fp4>::value;
  const int64_t slots = static_cast<int64_t>(sm_count()) * 8;
  const int64_t tokens = std::min<int64_t>(a.seqs.tokens, static_cast<int64_t>(a.seqs.batch) * a.seqs.max_new);
  const unsigned batch = static_cast<unsigned>(a.seqs.batch);
  const int ipr = a.head_dim / V;
  auto split = [&](int head0, int head1, int at_least) {
    HeadSplit s{};
    const int heads = head1 - head0;
    s.head0 = head0;
    s.head1 = head1;
    // a CTA of 256 threads holds whole heads
    s.passes = static_cast<int>(std::max<int64_t>(ceil_div(heads, 256 / ipr), std::min(at_least, heads)));
    s.per_pass = static_cast<int>(ceil_div(heads, s.passes));
    s.passes = static_cast<int>(ceil_div(heads, s.per_pass));
    s.tokens = std::max(1, 256 / (s.per_pass * ipr));
    return s;
  };
  auto threads = [&](const HeadSplit& s) { return static_cast<unsigned>(ceil_div(s.per_pass * ipr * s.tokens, 32) * 32); };
  // eight tokens or more for each place in a CTA, while that leaves enough CTAs
  auto walkers = [&](const HeadSplit& s) {
    const int64_t steps = ceil_div(a.seqs.max_new, s.tokens);
    return static_cast<unsigned>(std::min<int64_t>(steps, std::max<int64_t>(ceil_div(steps, 8), ceil_div(2 * slots, a.seqs.batch))));
  };
  const int heads = a.hq + 2 * a.hkv;
  a.all = split(0, heads, 3);
  if (tokens * a.all.passes <= slots) {
    // few tokens: one head of each thread per CTA, the shortest chain
    a.all.tokens = 1;
    launch_pdl(qkv_rotary_paged_kernel<T, KV, V, 1>,
               dim3(static_cast<unsigned>(a.seqs.max_new), batch, static_cast<unsigned>(a.all.passes)),
               dim3(threads(a.all)), 0, stream, a);
  } else if constexpr (kFp4) {
    a.q = split(0, a.hq, 4);
    a.kv = split(a.hq, heads, 2);
    launch_pdl(qkv_rotary_paged_fp4_kernel<T>, dim3(2u * std::max(walkers(a.q), walkers(a.kv)), batch),
               dim3(std::max(threads(a.q), threads(a.kv))), 0, stream, a);
  } else {
    a.all = split(0, heads, 5);
    launch_pdl(qkv_rotary_paged_kernel<T, KV, V, 5>, dim3(walkers(a.all), batch), dim3(threads(a.all)), 0, stream, a);
  }
}

// ---- gather ------------------------------------------------------------------------
struct GatherArgs {
  PagedSeqs seqs;  // positions: first rows (or null), starts: lengths (or null)
  const void* k_pages;
  const void* v_pages;
  void* k_out;
  void* v_out;
  float k_scale, v_scale;
  int hkv, head_dim;
  int64_t count;
};

constexpr int kGatherRows = 2;  // of a thread, in flight

// A thread owns elements [vi * V, vi * V + V) of a row and walks rows; grid = (row
// walkers, sequences x heads, K and V), no larger CTAs than the rows want. Bound by memory
// (the dense rows are written, and read from 16-bit pages, or from 4-bit ones a quarter of
// that) and by conversion: 16 ragged prompts of up to 2048 tokens, 4 heads of 128 out of
// 4-bit pages 21.6 us (four rows in flight 23.3, half the elements a thread 26 to 30); one
// row of 128 sequences, 8 heads, 2.9 us (4.7 with 256 threads a CTA).
template <typename T, typename KV, int V>
__global__ void __launch_bounds__(256) paged_gather_kernel(const GatherArgs a) {
  DLI_PDL_ENTRY();
  constexpr bool kFp4 = std::is_same<KV, Fp4>::value;
  constexpr int U = kGatherRows;
  const int b = blockIdx.y / a.hkv, h = blockIdx.y - b * a.hkv;
  const void* pages = blockIdx.z ? a.v_pages : a.k_pages;
  const float scale = blockIdx.z ? a.v_scale : a.k_scale;
  const int d = a.head_dim, ipr = d / V, page_rows = 1 << a.seqs.page_shift;
  const int per_cta = blockDim.x / ipr;  // rows
  const int vi = threadIdx.x % ipr, rl = threadIdx.x / ipr;
  if (rl >= per_cta) return;
  const int64_t rows_max = a.seqs.max_pages << a.seqs.page_shift;
  const int64_t first = a.seqs.positions ? min(a.seqs.positions[b], rows_max) : 0;
  int64_t end = a.seqs.starts ? a.seqs.starts[b] : rows_max;
  if (first < 0 || end > rows_max) {
    if (threadIdx.x == 0) set_device_error(a.seqs.err, kDevErrKvCapacity);
    end = min(end, rows_max);
  }
  T* out = static_cast<T*>(blockIdx.z ? a.v_out : a.k_out) + static_cast<int64_t>(blockIdx.y) * a.count * d + vi * V;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * per_cta;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * per_cta + rl; r0 < a.count; r0 += U * stride) {
    // all rows' pages, then all their bytes, then the stores
    int page[U], pr[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t p = first + r0 + k * stride;
      const bool there = r0 + k * stride < a.count && p >= 0 && p < end;
      pr[k] = static_cast<int>(p) & (page_rows - 1);
      page[k] = there ? page_of(a.seqs, b, static_cast<int>(p)) : -1;
    }
    Row<T, V> x[U];
    if constexpr (kFp4) {
      uint2 w[U];
      unsigned char sb[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        w[k] = make_uint2(0u, 0u);
        sb[k] = 0;
        if (page[k] >= 0) {
          const uint8_t* base = static_cast<const uint8_t*>(pages) + (static_cast<int64_t>(page[k]) * a.hkv + h) * fp4_block_bytes(page_rows, d);
          w[k] = *reinterpret_cast<const uint2*>(base + pr[k] * (d / 2) + vi * 8);
          sb[k] = base[page_rows * (d / 2) + pr[k] * (d / 16) + vi];
        }
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const float s = e4m3_value(sb[k]) * 16384.f;  // exact
#pragma unroll
        for (int j = 0; j < V; ++j) x[k].e[j] = from_f32<T>(e2m1_small(((j < 8 ? w[k].x : w[k].y) >> (4 * (j & 7))) & 15u) * s * scale);
      }
    } else {
#pragma unroll
      for (int k = 0; k < U; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) x[k].e[j] = from_f32<T>(0.f);
        if (page[k] >= 0) x[k].load(static_cast<const T*>(pages) + ((static_cast<int64_t>(page[k]) * a.hkv + h) * page_rows + pr[k]) * d + vi * V);
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (r0 + k * stride < a.count) x[k].store(out + (r0 + k * stride) * d);
  }
}

// ---- attention, any head dim up to 256, any type --------------------------------------
// One CTA per (packed row, query head), in fp32. Its warps take 32-key chunks in turn:
// lane j scores key j against the row's q (shared memory), the online softmax runs across
// the warp, and for O += p V each lane owns the elements lane, lane + 32, ...; the warps'
// (max, sum, O) are merged in order. It serves what the tensor-core kernels do not (other
// head dims, tensors off their alignment) and is bound by issue and by K and V rows that
// are fetched per query head: 8 x 1 token over 1000 keys, 16/4 heads of 80, bf16, 61 us
// (one warp per row and head 476 us), of 256 114 us, 4-bit pages of 96 84 us.
constexpr int kGeneralWarps = 8;

// sum of q[c] * K[c] over the row pr of a block at `block` (of one head of a page)
template <typename T, typename KV>
__device__ __forceinline__ float general_dot(const float* sq, const void* pages, int64_t block, int page_rows, int d, int pr,
                                             bool vec) {
  float dot = 0.f;
  if constexpr (std::is_same<KV, Fp4>::value) {
    const uint8_t* base = static_cast<const uint8_t*>(pages) + block * fp4_block_bytes(page_rows, d);
    for (int c = 0; c < d; c += 16) {
      const uint2 w = *reinterpret_cast<const uint2*>(base + pr * (d / 2) + c / 2);
      const float s = e4m3_value(base[page_rows * (d / 2) + pr * (d / 16) + c / 16]) * 16384.f;
      float part = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) part = fmaf(sq[c + j], e2m1_small(((j < 8 ? w.x : w.y) >> (4 * (j & 7))) & 15u), part);
      dot = fmaf(part, s, dot);
    }
  } else {
    const T* k = static_cast<const T*>(pages) + (block * page_rows + pr) * d;
    int c = 0;
    if (vec) {
      constexpr int N = Vec16<T>::N;
#pragma unroll 4
      for (; c + N <= d; c += N) {
        const Vec16<T> v = load16(k + c);
#pragma unroll
        for (int j = 0; j < N; ++j) dot = fmaf(sq[c + j], to_f32(v.e[j]), dot);
      }
    }
    for (; c < d; ++c) dot = fmaf(sq[c], to_f32(k[c]), dot);
  }
  return dot;
}

template <typename T, typename KV>
__global__ void __launch_bounds__(32 * kGeneralWarps) attn_paged_general_kernel(const PagedAttnArgs a, bool vec) {
  DLI_PDL_ENTRY();
  constexpr bool kFp4 = std::is_same<KV, Fp4>::value;
  constexpr int W = kGeneralWarps;
  extern __shared__ float general_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.y, d = a.head_dim;
  float* sq = general_smem;  // [d]
  float* so = sq + d;        // [W][d]
  float* sm = so + W * d;    // [W], then the sums [W]
  const SeqRows sr = seq_rows(a.seqs, b, threadIdx.x == 0 && blockIdx.x == 0);
  const int page_rows = 1 << a.seqs.page_shift;
  for (int64_t i = blockIdx.x; i < static_cast<int64_t>(sr.n) * a.hq; i += gridDim.x) {
    const int t = static_cast<int>(i / a.hq), h = static_cast<int>(i - static_cast<int64_t>(t) * a.hq);
    const int kvh = h / a.group, pos = sr.past + t;
    const int64_t at = ((sr.row0 + t) * a.hq + h) * d;
    __syncthreads();
    for (int c = threadIdx.x; c < d; c += 32 * W) sq[c] = to_f32(static_cast<const T*>(a.q)[at + c]);
    __syncthreads();
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const int key_lo = max(0, pos - a.window + 1);
    for (int j0 = key_lo + 32 * warp; j0 <= pos; j0 += 32 * W) {
      const int j = j0 + lane;
      float x = -INFINITY;
      int64_t row = -1;  // (page, head) block of this lane's key
      int pr = 0;
      if (j <= pos) {
        const int page = page_of(a.seqs, b, j);
        pr = j & (page_rows - 1);
        float dot = 0.f;
        if (page >= 0) {
          row = static_cast<int64_t>(page) * a.hkv + kvh;
          dot = general_dot<T, KV>(sq, a.k_pages, row, page_rows, d, pr, vec);
        }
        x = dot * a.scale;
        if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
        x += slope * static_cast<float>(j - pos);
      }
      const float m_new = fmaxf(m, warp_max(x));
      const float p = j <= pos ? expf(x - m_new) : 0.f;
      const float alpha = m == -INFINITY ? 0.f : expf(m - m_new);
      l = l * alpha + warp_sum(p);
      m = m_new;
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] *= alpha;
      const int keys = min(32, pos + 1 - j0);
#pragma unroll 4
      for (int k = 0; k < keys; ++k) {
        const float pk = __shfl_sync(0xffffffffu, p, k);
        const int64_t rk = __shfl_sync(0xffffffffu, row, k);
        const int prk = __shfl_sync(0xffffffffu, pr, k);
        if (rk < 0) continue;
        if constexpr (kFp4) {
          const uint8_t* base = static_cast<const uint8_t*>(a.v_pages) + rk * fp4_block_bytes(page_rows, d);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (lane + 32 * e < d) o[e] = fmaf(pk, fp4_element(base, page_rows, d, prk, lane + 32 * e), o[e]);
        } else {
          const T* v = static_cast<const T*>(a.v_pages) + (rk * page_rows + prk) * d;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (lane + 32 * e < d) o[e] = fmaf(pk, to_f32(v[lane + 32 * e]), o[e]);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (lane + 32 * e < d) so[warp * d + lane + 32 * e] = o[e];
    if (lane == 0) {
      sm[warp] = m;
      sm[W + warp] = l;
    }
    __syncthreads();
    // a warp without keys has m = -inf, l = 0 and O = 0
    float top = sm[0], sum = 0.f, w[W];
#pragma unroll
    for (int k = 1; k < W; ++k) top = sm[k] > top || isnan(sm[k]) ? sm[k] : top;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      w[k] = sm[W + k] == 0.f ? 0.f : expf(sm[k] - top);
      sum += sm[W + k] * w[k];
    }
    const float inv = a.v_scale / sum;
    for (int c = threadIdx.x; c < d; c += 32 * W) {
      float x = 0.f;
#pragma unroll
      for (int k = 0; k < W; ++k) x = fmaf(so[k * d + c], w[k], x);
      static_cast<T*>(a.out)[at + c] = from_f32<T>(x * inv);
    }
  }
}

template <typename T, typename KV>
dli_status launch_attn_general(const PagedAttnArgs& a, cudaStream_t stream) {
  const int64_t per_seq = static_cast<int64_t>(a.seqs.max_new) * a.hq;
  const int64_t walkers = std::min<int64_t>(per_seq, std::max<int64_t>(1, ceil_div(64ll * sm_count(), a.seqs.batch)));
  const bool vec = a.head_dim % Vec16<T>::N == 0 && aligned(a.k_pages, 16);
  launch_pdl(attn_paged_general_kernel<T, KV>,
             dim3(static_cast<unsigned>(walkers), static_cast<unsigned>(a.seqs.batch)), dim3(32 * kGeneralWarps),
             ((kGeneralWarps + 1) * a.head_dim + 2 * kGeneralWarps) * sizeof(float), stream, a, vec);
  return check_launch("attention_paged");
}

// Calls of the decode kernel (the others go to the tcgen05 kernel): float32, more heads
// per KV head than a tcgen05 tile has rows, and up to 16 query rows per KV head over
// 16-bit pages or 32 over 4-bit ones, which the tcgen05 kernel has to convert. us, decode
// | tcgen05, over 1 x 30,000 keys and 32 x 2,304: 14 rows 28 | 35 and 30 | 36; 28 rows
// 33 | 35 and 38 | 35; 32 rows 48 | 38 and 65 | 53; 4 bits: 28 rows 32 | 38 and 43 | 43;
// 56 rows 48 | 38 and 73 | 45.
bool few_rows(dli_dtype dtype, bool fp4, int64_t group, int64_t max_new) {
  return dtype == DLI_DTYPE_F32 || group > 128 || group * max_new <= (fp4 ? 32 : 16);
}

// ---- argument checks -----------------------------------------------------------------
int page_shift_of(int64_t page_size) {
  for (int s = 4; s <= 7; ++s)
    if (page_size == (1ll << s)) return s;
  return -1;
}

dli_status check_pages(const std::string& what, int64_t batch, int64_t kv_heads, int64_t head_dim, int64_t page_size,
                       int64_t num_pages, int64_t max_pages, float k_scale, float v_scale, dli_dtype dtype,
                       dli_dtype kv_dtype, const void* k_pages, const void* v_pages, const void* page_table) {
  if (batch < 0 || kv_heads <= 0 || head_dim <= 0 || num_pages < 0 || max_pages < 0)
    return fail(DLI_ERR_INVALID_ARGUMENT, what + ": bad sizes");
  if (page_shift_of(page_size) < 0)
    return fail(DLI_ERR_INVALID_ARGUMENT, what + ": page_size must be 16, 32, 64 or 128");
  if (!is_float_dtype(dtype)) return fail(DLI_ERR_INVALID_ARGUMENT, what + " expects a float32/bfloat16/float16 dtype");
  if (kv_dtype != dtype && kv_dtype != DLI_DTYPE_FP4)
    return fail(DLI_ERR_INVALID_ARGUMENT, what + ": kv_dtype must be dtype or FP4");
  if (kv_dtype == DLI_DTYPE_FP4) {
    if (head_dim % 16 != 0) return fail(DLI_ERR_INVALID_ARGUMENT, what + ": 4-bit pages need head_dim % 16 == 0");
    if (!(k_scale > 0.f) || !(v_scale > 0.f) || std::isinf(k_scale) || std::isinf(v_scale))
      return fail(DLI_ERR_INVALID_ARGUMENT, what + ": k_scale and v_scale must be positive and finite");
    if (!aligned(k_pages, 16) || !aligned(v_pages, 16))
      return fail(DLI_ERR_INVALID_ARGUMENT, what + ": 4-bit pages must be 16-byte aligned");
  }
  if (batch > 65535 || kv_heads > 65535) return fail(DLI_ERR_UNSUPPORTED, what + ": more than 65535 sequences or heads");
  if (num_pages > INT_MAX || max_pages > (1ll << 30) / page_size)
    return fail(DLI_ERR_UNSUPPORTED, what + ": more than 2^30 rows per sequence or 2^31 pages");
  // the kernels look rows up in the table before they compare its entries with num_pages
  if (batch > 0 && max_pages > 0 && (page_table == nullptr || (num_pages > 0 && (k_pages == nullptr || v_pages == nullptr))))
    return fail(DLI_ERR_INVALID_ARGUMENT, what + ": pages and page_table required");
  return DLI_OK;
}

dli_status check_rows(const std::string& what, int64_t tokens, int64_t batch, int64_t max_new, int64_t q_heads,
                      const void* positions, const void* starts) {
  if (tokens < 0 || max_new < 0 || q_heads <= 0) return fail(DLI_ERR_INVALID_ARGUMENT, what + ": bad sizes");
  if (positions == nullptr) return fail(DLI_ERR_INVALID_ARGUMENT, what + ": positions required");
  if (q_heads > 65535) return fail(DLI_ERR_UNSUPPORTED, what + ": more than 65535 heads");
  if (max_new > (1 << 30)) return fail(DLI_ERR_UNSUPPORTED, what + ": sequence too long");
  if (starts == nullptr && tokens < batch * max_new)
    return fail(DLI_ERR_INVALID_ARGUMENT, what + ": fewer rows than batch * max_new");
  return DLI_OK;
}

PagedSeqs make_seqs(const int64_t* positions, const int64_t* starts, const int32_t* page_table, int64_t tokens,
                    int64_t batch, int64_t max_new, int64_t page_size, int64_t num_pages, int64_t max_pages) {
  PagedSeqs s{};
  s.positions = positions;
  s.starts = starts;
  s.page_table = page_table;
  s.tokens = tokens;
  s.num_pages = num_pages;
  s.max_pages = max_pages;
  s.batch = static_cast<int>(batch);
  s.max_new = static_cast<int>(std::min(max_new, tokens));  // no sequence has more rows than there are
  s.page_shift = page_shift_of(page_size);
  s.err = device_error_word();
  return s;
}

}  // namespace
}  // namespace dli_sm100

using namespace dli_sm100;

extern "C" size_t dli_sm100_paged_kv_page_bytes(int64_t kv_heads, int64_t page_size, int64_t head_dim,
                                                dli_dtype kv_dtype) {
  if (kv_heads <= 0 || head_dim <= 0 || page_shift_of(page_size) < 0) return 0;
  if (kv_dtype == DLI_DTYPE_FP4)
    return head_dim % 16 == 0 ? static_cast<size_t>(kv_heads * fp4_block_bytes(page_size, head_dim)) : 0;
  if (!is_float_dtype(kv_dtype)) return 0;
  return static_cast<size_t>(kv_heads * page_size * head_dim) * dtype_bytes(kv_dtype);
}

extern "C" dli_status dli_sm100_qkv_rotary_paged(const void* qkv, const float* cos_table, const float* sin_table,
                                                 const int64_t* positions, const int64_t* starts,
                                                 const int32_t* page_table, void* q_out, void* k_pages,
                                                 void* v_pages, int64_t tokens, int64_t batch, int64_t max_new,
                                                 int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                                 int64_t pairs, int64_t table_rows, int64_t page_size,
                                                 int64_t num_pages, int64_t max_pages, float k_scale,
                                                 float v_scale, dli_dtype dtype, dli_dtype kv_dtype,
                                                 void* stream) {
  const char* what = "qkv_rotary_paged";
  dli_status st = check_pages(what, batch, kv_heads, head_dim, page_size, num_pages, max_pages, k_scale, v_scale,
                              dtype, kv_dtype, k_pages, v_pages, page_table);
  if (st != DLI_OK) return st;
  st = check_rows(what, tokens, batch, max_new, q_heads, positions, starts);
  if (st != DLI_OK) return st;
  if (head_dim % 2 != 0 || pairs < 0 || 2 * pairs > head_dim || table_rows < 0)
    return fail(DLI_ERR_INVALID_ARGUMENT, "qkv_rotary_paged: bad head_dim/pairs");
  if (batch == 0 || max_new == 0 || tokens == 0) return ok();
  AppendArgs a{};
  a.seqs = make_seqs(positions, starts, page_table, tokens, batch, max_new, page_size, num_pages, max_pages);
  a.qkv = qkv;
  a.cos_t = cos_table;
  a.sin_t = sin_table;
  a.q_out = q_out;
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.hq = static_cast<int>(q_heads);
  a.hkv = static_cast<int>(kv_heads);
  a.head_dim = static_cast<int>(head_dim);
  a.pairs = static_cast<int>(pairs);
  a.table_rows = table_rows;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  const bool al = aligned(qkv, 16) && aligned(q_out, 16) && aligned(k_pages, 16) && aligned(v_pages, 16);
  if (kv_dtype == DLI_DTYPE_FP4 && !al)
    return fail(DLI_ERR_INVALID_ARGUMENT, "qkv_rotary_paged: 4-bit pages need 16-byte aligned tensors");
  if (head_dim > 256) return fail(DLI_ERR_UNSUPPORTED, "qkv_rotary_paged: head_dim > 256");
  a.vec_tables = pairs % 4 == 0 && aligned(cos_table, 16) && aligned(sin_table, 16);
  st = dispatch_float(dtype, what, [&](auto tag) {
    using T = decltype(tag);
    constexpr int V = Vec16<T>::N;
    if (kv_dtype == DLI_DTYPE_FP4) launch_append<T, Fp4, 8>(a, as_stream(stream));
    else if (al && head_dim % V == 0) launch_append<T, T, V>(a, as_stream(stream));
    else launch_append<T, T, 2>(a, as_stream(stream));
  });
  if (st != DLI_OK) return st;
  return check_launch(what);
}

extern "C" dli_status dli_sm100_paged_gather(const void* k_pages, const void* v_pages, const int32_t* page_table,
                                             const int64_t* first, const int64_t* lengths, void* k_out, void* v_out,
                                             int64_t batch, int64_t count, int64_t kv_heads, int64_t head_dim,
                                             int64_t page_size, int64_t num_pages, int64_t max_pages, float k_scale,
                                             float v_scale, dli_dtype dtype, dli_dtype kv_dtype, void* stream) {
  const char* what = "paged_gather";
  dli_status st = check_pages(what, batch, kv_heads, head_dim, page_size, num_pages, max_pages, k_scale, v_scale,
                              dtype, kv_dtype, k_pages, v_pages, page_table);
  if (st != DLI_OK) return st;
  if (count < 0 || count > (1ll << 30)) return fail(DLI_ERR_INVALID_ARGUMENT, "paged_gather: bad count");
  if (batch * kv_heads > 65535) return fail(DLI_ERR_UNSUPPORTED, "paged_gather: batch * kv_heads > 65535");
  if (batch == 0 || count == 0) return ok();
  GatherArgs a{};
  a.seqs = make_seqs(first, lengths, page_table, 0, batch, 0, page_size, num_pages, max_pages);
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.k_out = k_out;
  a.v_out = v_out;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.hkv = static_cast<int>(kv_heads);
  a.head_dim = static_cast<int>(head_dim);
  a.count = count;
  const bool al = aligned(k_pages, 16) && aligned(v_pages, 16) && aligned(k_out, 16) && aligned(v_out, 16);
  if (kv_dtype == DLI_DTYPE_FP4 && !al)
    return fail(DLI_ERR_INVALID_ARGUMENT, "paged_gather: 4-bit pages need 16-byte aligned tensors");
  if (head_dim > 256) return fail(DLI_ERR_UNSUPPORTED, "paged_gather: head_dim > 256");
  st = dispatch_float(dtype, what, [&](auto tag) {
    using T = decltype(tag);
    auto launch = [&](auto kernel, int64_t elements) {  // of a thread
      // no more threads than the rows want
      const int64_t per_row = head_dim / elements, threads = std::max<int64_t>(per_row, std::min<int64_t>(256, count * per_row));
      const int64_t per_cta = std::min<int64_t>(256, ceil_div(threads, 32) * 32) / per_row;
      const int64_t walkers = std::min<int64_t>(ceil_div(count, kGatherRows * per_cta),
                                                std::max<int64_t>(1, ceil_div(32ll * sm_count(), batch * kv_heads)));
      launch_pdl(kernel, dim3(static_cast<unsigned>(walkers), static_cast<unsigned>(batch * kv_heads), 2u),
                 dim3(static_cast<unsigned>(std::min<int64_t>(256, ceil_div(threads, 32) * 32))), 0, as_stream(stream), a);
    };
    if (kv_dtype == DLI_DTYPE_FP4) launch(paged_gather_kernel<T, Fp4, 16>, 16);
    else if (al && head_dim % Vec16<T>::N == 0) launch(paged_gather_kernel<T, T, Vec16<T>::N>, Vec16<T>::N);
    else launch(paged_gather_kernel<T, T, 1>, 1);
  });
  if (st != DLI_OK) return st;
  return check_launch(what);
}

extern "C" size_t dli_sm100_attention_paged_workspace_size(int64_t tokens, int64_t batch, int64_t max_new,
                                                           int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                                           int64_t page_size, int64_t max_pages, dli_dtype dtype,
                                                           dli_dtype kv_dtype) {
  if (tokens <= 0 || batch <= 0 || max_new <= 0 || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads != 0) return 0;
  if (page_shift_of(page_size) < 0 || max_pages <= 0 || max_pages > (1ll << 30) / page_size) return 0;
  if (!is_float_dtype(dtype) || (head_dim != 64 && head_dim != 128)) return 0;
  max_new = std::min(max_new, tokens);
  const int64_t group = q_heads / kv_heads, max_keys = max_pages * page_size;
  if (few_rows(dtype, kv_dtype == DLI_DTYPE_FP4, group, max_new)) return paged_decode_workspace(batch, kv_heads, group, max_new, head_dim, max_keys, dtype);
  return paged_prefill_workspace(batch, kv_heads, group, max_new, head_dim, max_keys);
}

extern "C" dli_status dli_sm100_attention_paged(const void* q, const void* k_pages, const void* v_pages,
                                                const int64_t* positions, const int64_t* starts,
                                                const int32_t* page_table, const float* slopes, void* out,
                                                int64_t tokens, int64_t batch, int64_t max_new, int64_t q_heads,
                                                int64_t kv_heads, int64_t head_dim, int64_t page_size,
                                                int64_t num_pages, int64_t max_pages, float scale, float softcap,
                                                int64_t window, float k_scale, float v_scale, dli_dtype dtype,
                                                dli_dtype kv_dtype, void* workspace, size_t workspace_bytes,
                                                void* stream) {
  const char* what = "attention_paged";
  dli_status st = check_pages(what, batch, kv_heads, head_dim, page_size, num_pages, max_pages, k_scale, v_scale,
                              dtype, kv_dtype, k_pages, v_pages, page_table);
  if (st != DLI_OK) return st;
  st = check_rows(what, tokens, batch, max_new, q_heads, positions, starts);
  if (st != DLI_OK) return st;
  if (q_heads % kv_heads != 0)
    return fail(DLI_ERR_INVALID_ARGUMENT, "attention_paged: q heads must be a multiple of kv heads");
  if (!(softcap >= 0.f) || std::isinf(softcap) || std::isnan(scale) || std::isinf(scale) || window < 0)
    return fail(DLI_ERR_INVALID_ARGUMENT, "attention_paged: softcap and window must not be negative, scale finite");
  if (head_dim > 256) return fail(DLI_ERR_UNSUPPORTED, "attention_paged: head_dim > 256");
  if (batch == 0 || max_new == 0 || tokens == 0) return ok();
  PagedAttnArgs a{};
  a.seqs = make_seqs(positions, starts, page_table, tokens, batch, max_new, page_size, num_pages, max_pages);
  a.q = q;
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.slopes = slopes;
  a.out = out;
  a.hq = static_cast<int>(q_heads);
  a.hkv = static_cast<int>(kv_heads);
  a.group = static_cast<int>(q_heads / kv_heads);
  a.head_dim = static_cast<int>(head_dim);
  a.window = window > 0 && window < INT_MAX ? static_cast<int>(window) : INT_MAX;
  const bool fp4 = kv_dtype == DLI_DTYPE_FP4;
  a.scale = (scale > 0.f ? scale : 1.0f / sqrtf(static_cast<float>(head_dim))) * (fp4 ? k_scale : 1.f);
  // caps beyond 2^64 or below 2^-64 bend nothing more (scores past 2^51 keep one key, those
  // within 2^-64 weigh all alike), and their reciprocals stay normal
  a.softcap = softcap > 0.f ? std::max(std::min(softcap, 0x1p64f), 0x1p-64f) : 0.f;
  a.v_scale = fp4 ? v_scale : 1.f;
  if (few_rows(dtype, fp4, a.group, a.seqs.max_new)) {
    if (paged_decode_serves(a, dtype)) return run_paged_decode(a, dtype, kv_dtype, workspace, workspace_bytes, as_stream(stream));
  } else if (paged_prefill_serves(a, dtype, kv_dtype)) {
    return run_paged_prefill(a, dtype, kv_dtype, workspace, workspace_bytes, as_stream(stream));
  }
  dli_status run = DLI_OK;
  st = dispatch_float(dtype, what, [&](auto tag) {
    using T = decltype(tag);
    run = fp4 ? launch_attn_general<T, Fp4>(a, as_stream(stream)) : launch_attn_general<T, T>(a, as_stream(stream));
  });
  return st != DLI_OK ? st : run;
}
