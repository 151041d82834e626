// Paged KV cache: the append with rotary embedding, the gather of cached rows,
// and the entry points of the attention over pages with its general kernel.
//
// Pages are [num_pages, Hkv, page_size, D] of the model's type, or 4-bit: per
// (page, head) the rows' E2M1 codes, then their E4M3 scales, one per 16 elements.
#include <algorithm>
#include <climits>
#include <cmath>

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
// most 7 bits, so the comparisons decide as the exact value would.
__device__ __forceinline__ unsigned e4m3_scale(float most) {
  unsigned c = __nv_cvt_float_to_fp8(most * (1.f / 6.f), __NV_SATFINITE, __NV_E4M3);
  const float v = e4m3_value(c);
  if (c < 126u) {
    const float up = 3.f * (v + e4m3_value(c + 1u));
    if (most > up || (most == up && (c & 1u))) return c + 1u;
  }
  if (c > 0u) {
    const float down = 3.f * (v + e4m3_value(c - 1u));
    if (most < down || (most == down && (c & 1u))) return c - 1u;
  }
  return c;
}

// 16 values (rounded to odd where they are not exact) -> scale byte and 8 code
// bytes. A value's code is the number of rounding borders below it: 0.25, 0.75,
// ... times the scale, products of 3-bit numbers, hence exact; a border itself
// goes to the even code.
__device__ __forceinline__ void fp4_block(const float (&x)[16], unsigned& scale, uint2& codes) {
  float most = 0.f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    most = fmaxf(most, fabsf(x[i]));
    nan |= x[i] != x[i];
  }
  scale = nan ? 0x7Fu : e4m3_scale(most);
  const float s = nan ? 0.f : e4m3_value(scale);
  unsigned w[2] = {0u, 0u};
  if (s > 0.f) {
    const float b0 = 0.25f * s, b1 = 0.75f * s, b2 = 1.25f * s, b3 = 1.75f * s, b4 = 2.5f * s, b5 = 3.5f * s,
                b6 = 5.f * s;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float a = fabsf(x[i]);
      unsigned c = static_cast<unsigned>(a > b0) + static_cast<unsigned>(a >= b1) + static_cast<unsigned>(a > b2) +
                   static_cast<unsigned>(a >= b3) + static_cast<unsigned>(a > b4) + static_cast<unsigned>(a >= b5) +
                   static_cast<unsigned>(a > b6);
      if (x[i] < 0.f) c |= 8u;
      w[i / 8] |= c << (4 * (i % 8));
    }
  }
  codes = make_uint2(w[0], w[1]);
}

// ---- append ------------------------------------------------------------------------
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
  int heads_per_pass, passes;
};

// A thread owns elements [vi * V, vi * V + V) of a head row and walks heads
// hl, hl + heads_per_pass, ... of its token: the token's cos/sin values are read
// once for all of them. grid = (token walkers, sequences, parts of the head
// passes). Bound by memory: it reads qkv once and writes q, k and v once.
template <typename T, typename KV, int V>
__global__ void __launch_bounds__(256) qkv_rotary_paged_kernel(const AppendArgs a) {
  DLI_PDL_ENTRY();
  constexpr bool kFp4 = std::is_same<KV, Fp4>::value;
  constexpr int kVec = V * static_cast<int>(sizeof(T)) / 16;  // 16-byte vectors per item, 0: one pair
  const int b = blockIdx.y;
  const int d = a.head_dim, ipr = d / V, heads = a.hq + 2 * a.hkv;
  const int vi = threadIdx.x % ipr, hl = threadIdx.x / ipr;
  if (hl >= a.heads_per_pass) return;
  const SeqRows sr = seq_rows(a.seqs, b, true);
  const int page_rows = 1 << a.seqs.page_shift;
  const int part = static_cast<int>(gridDim.z);
  for (int t = blockIdx.x; t < sr.n; t += gridDim.x) {
    const int p = sr.past + t;
    const int64_t row = sr.row0 + t;
    float c[V / 2], s[V / 2];
    const int first_pair = vi * (V / 2);
    const bool in_table = p < a.table_rows;
    if (!in_table && first_pair < a.pairs) set_device_error(a.seqs.err, kDevErrRotaryPosition);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      c[j] = s[j] = 0.f;
      if (in_table && first_pair + j < a.pairs) {
        c[j] = a.cos_t[static_cast<int64_t>(p) * a.pairs + first_pair + j];
        s[j] = a.sin_t[static_cast<int64_t>(p) * a.pairs + first_pair + j];
      }
    }
    const int page = page_of(a.seqs, b, p);
    for (int pass = blockIdx.z; pass < a.passes; pass += part) {
      const int h = hl + pass * a.heads_per_pass;
      if (h >= heads) break;
      float x[V];
      const T* src = static_cast<const T*>(a.qkv) + (row * heads + h) * d + vi * V;
      if constexpr (kVec > 0) {
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
          const Vec16<T> in = load16(src + v * Vec16<T>::N);
#pragma unroll
          for (int j = 0; j < Vec16<T>::N; ++j) x[v * Vec16<T>::N + j] = to_f32(in.e[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = to_f32(src[j]);
      }
      T* dst = nullptr;
      if (h < a.hq) {
        dst = static_cast<T*>(a.q_out) + (row * a.hq + h) * d + vi * V;
      } else {
        if (page < 0) continue;
        const bool is_k = h < a.hq + a.hkv;
        const int kvh = is_k ? h - a.hq : h - a.hq - a.hkv;
        const int64_t block = static_cast<int64_t>(page) * a.hkv + kvh;
        const int r = p & (page_rows - 1);
        void* pages = is_k ? a.k_pages : a.v_pages;
        if constexpr (kFp4) {
          const float cache_scale = is_k ? a.k_scale : a.v_scale;
          if (is_k || cache_scale != 1.f) {
            // products of a 24-bit and an at most 24-bit number are exact in 53 bits
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
              double u = x[2 * j], w = x[2 * j + 1];
              if (is_k && in_table && first_pair + j < a.pairs) {
                const double cd = c[j], sd = s[j];
                const double u0 = u * cd - w * sd;
                w = u * sd + w * cd;
                u = u0;
              }
              if (cache_scale != 1.f) {
                u /= static_cast<double>(cache_scale);
                w /= static_cast<double>(cache_scale);
              }
              x[2 * j] = round_to_odd(u);
              x[2 * j + 1] = round_to_odd(w);
            }
          }
          unsigned scale;
          uint2 codes;
          fp4_block(x, scale, codes);
          uint8_t* base = static_cast<uint8_t*>(pages) + block * fp4_block_bytes(page_rows, d);
          *reinterpret_cast<uint2*>(base + r * (d / 2) + vi * 8) = codes;
          base[page_rows * (d / 2) + r * (d / 16) + vi] = static_cast<uint8_t>(scale);
          continue;
        }
        dst = static_cast<T*>(pages) + (block * page_rows + r) * d + vi * V;
        if (!is_k) {  // v is copied
          if constexpr (kVec > 0) {
#pragma unroll
            for (int v = 0; v < kVec; ++v) store16(dst + v * Vec16<T>::N, load16(src + v * Vec16<T>::N));
          } else {
#pragma unroll
            for (int j = 0; j < V; ++j) dst[j] = src[j];
          }
          continue;
        }
      }
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        const float u = x[2 * j], w = x[2 * j + 1];
        if (in_table && first_pair + j < a.pairs) {
          x[2 * j] = u * c[j] - w * s[j];
          x[2 * j + 1] = u * s[j] + w * c[j];
        }
      }
      if constexpr (kVec > 0) {
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
          Vec16<T> o;
#pragma unroll
          for (int j = 0; j < Vec16<T>::N; ++j) o.e[j] = from_f32<T>(x[v * Vec16<T>::N + j]);
          store16(dst + v * Vec16<T>::N, o);
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) dst[j] = from_f32<T>(x[j]);
      }
    }
  }
}

template <typename T, typename KV, int V>
void launch_append(AppendArgs a, cudaStream_t stream) {
  const int ipr = a.head_dim / V, heads = a.hq + 2 * a.hkv;
  a.passes = static_cast<int>(ceil_div(static_cast<int64_t>(heads) * ipr, 256));
  a.heads_per_pass = static_cast<int>(ceil_div(heads, a.passes));
  const int threads = std::min(256, static_cast<int>(ceil_div(a.heads_per_pass * ipr, 32)) * 32);
  // few tokens: one head pass per CTA, the shortest chain; many: all passes in one
  const int64_t slots = static_cast<int64_t>(sm_count()) * 8;
  const int64_t tokens = static_cast<int64_t>(a.seqs.batch) * a.seqs.max_new;
  const unsigned parts = tokens * a.passes <= slots ? static_cast<unsigned>(a.passes) : 1u;
  const int64_t walkers = std::min<int64_t>(a.seqs.max_new, ceil_div(4 * slots, a.seqs.batch));
  launch_pdl(qkv_rotary_paged_kernel<T, KV, V>,
             dim3(static_cast<unsigned>(walkers), static_cast<unsigned>(a.seqs.batch), parts),
             dim3(static_cast<unsigned>(threads)), 0, stream, a);
}

// ---- gather ------------------------------------------------------------------------
struct GatherArgs {
  PagedSeqs seqs;  // positions: first rows (or null), starts: lengths (or null)
  const void* pages[2];
  void* out[2];
  float scale[2];
  int hkv, head_dim;
  int64_t count;
};

// One thread per 8 elements (one in the general form) of an output row; grid =
// (row walkers, sequences x heads, K and V). Bound by memory.
template <typename T, typename KV, int V>
__global__ void __launch_bounds__(256) paged_gather_kernel(const GatherArgs a) {
  DLI_PDL_ENTRY();
  constexpr bool kFp4 = std::is_same<KV, Fp4>::value;
  const int b = blockIdx.y / a.hkv, h = blockIdx.y - b * a.hkv;
  const int which = blockIdx.z;
  const int d = a.head_dim, ipr = d / V, page_rows = 1 << a.seqs.page_shift;
  const int64_t rows_max = a.seqs.max_pages << a.seqs.page_shift;
  const int64_t first = a.seqs.positions ? a.seqs.positions[b] : 0;
  int64_t end = a.seqs.starts ? a.seqs.starts[b] : rows_max;
  if (first < 0 || end > rows_max) {
    if (threadIdx.x == 0) set_device_error(a.seqs.err, kDevErrKvCapacity);
    end = min(end, rows_max);
  }
  T* out = static_cast<T*>(a.out[which]) + static_cast<int64_t>(blockIdx.y) * a.count * d;
  const int64_t items = a.count * ipr;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < items; i += gridDim.x * 256ll) {
    const int64_t r = i / ipr;
    const int c = static_cast<int>(i - r * ipr) * V;
    const int64_t p = first + r;
    T v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = from_f32<T>(0.f);
    const int page = (p >= 0 && p < end) ? page_of(a.seqs, b, static_cast<int>(p)) : -1;
    if (page >= 0) {
      const int64_t block = static_cast<int64_t>(page) * a.hkv + h;
      const int pr = static_cast<int>(p) & (page_rows - 1);
      if constexpr (kFp4) {
        const uint8_t* base = static_cast<const uint8_t*>(a.pages[which]) + block * fp4_block_bytes(page_rows, d);
        const float s = e4m3_value(base[page_rows * (d / 2) + pr * (d / 16) + c / 16]);
        const uint32_t w = *reinterpret_cast<const uint32_t*>(base + pr * (d / 2) + c / 2);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = from_f32<T>(e2m1_value((w >> (4 * j)) & 15u) * s * a.scale[which]);
      } else {
        const T* src = static_cast<const T*>(a.pages[which]) + (block * page_rows + pr) * d + c;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = src[j];
      }
    }
    T* dst = out + r * d + c;
    if constexpr (V * sizeof(T) >= 16) {
#pragma unroll
      for (int q = 0; q < static_cast<int>(V * sizeof(T) / 16); ++q)
        *reinterpret_cast<uint4*>(dst + q * Vec16<T>::N) = *reinterpret_cast<uint4*>(&v[q * Vec16<T>::N]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) dst[j] = v[j];
    }
  }
}

// ---- attention, any head dim up to 256, any type --------------------------------------
// One warp per (packed row, query head): lane j scores key j of a 32-key chunk
// against the row's q (shared memory), the online softmax runs across the warp,
// and for O += p V each lane owns the elements lane, lane + 32, ... In fp32.
template <typename T, typename KV>
__global__ void __launch_bounds__(128) attn_paged_general_kernel(const PagedAttnArgs a) {
  DLI_PDL_ENTRY();
  constexpr bool kFp4 = std::is_same<KV, Fp4>::value;
  extern __shared__ float sq_all[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.y, d = a.head_dim;
  const SeqRows sr = seq_rows(a.seqs, b, threadIdx.x == 0);
  const int page_rows = 1 << a.seqs.page_shift;
  float* sq = sq_all + warp * d;
  for (int64_t i = blockIdx.x * 4ll + warp; i < static_cast<int64_t>(sr.n) * a.hq; i += gridDim.x * 4ll) {
    const int t = static_cast<int>(i / a.hq), h = static_cast<int>(i - static_cast<int64_t>(t) * a.hq);
    const int kvh = h / a.group, pos = sr.past + t;
    const int64_t at = ((sr.row0 + t) * a.hq + h) * d;
    __syncwarp();
    for (int c = lane; c < d; c += 32) sq[c] = to_f32(static_cast<const T*>(a.q)[at + c]);
    __syncwarp();
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const int key_lo = max(0, pos - a.window + 1);
    for (int j0 = key_lo; j0 <= pos; j0 += 32) {
      const int j = j0 + lane;
      float x = -INFINITY;
      int64_t row = -1;  // element (or byte block) index of this lane's key row
      int pr = 0;
      if (j <= pos) {
        const int page = page_of(a.seqs, b, j);
        pr = j & (page_rows - 1);
        float dot = 0.f;
        if (page >= 0) {
          row = static_cast<int64_t>(page) * a.hkv + kvh;
          if constexpr (kFp4) {
            const uint8_t* base = static_cast<const uint8_t*>(a.k_pages) + row * fp4_block_bytes(page_rows, d);
            for (int c = 0; c < d; ++c) dot = fmaf(sq[c], fp4_element(base, page_rows, d, pr, c), dot);
          } else {
            const T* k = static_cast<const T*>(a.k_pages) + (row * page_rows + pr) * d;
            for (int c = 0; c < d; ++c) dot = fmaf(sq[c], to_f32(k[c]), dot);
          }
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
    const float inv = a.v_scale / l;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (lane + 32 * e < d) static_cast<T*>(a.out)[at + lane + 32 * e] = from_f32<T>(o[e] * inv);
  }
}

template <typename T, typename KV>
dli_status launch_attn_general(const PagedAttnArgs& a, cudaStream_t stream) {
  const int64_t per_seq = ceil_div(static_cast<int64_t>(a.seqs.max_new) * a.hq, 4);
  const int64_t walkers = std::min<int64_t>(per_seq, std::max<int64_t>(1, ceil_div(64ll * sm_count(), a.seqs.batch)));
  launch_pdl(attn_paged_general_kernel<T, KV>,
             dim3(static_cast<unsigned>(walkers), static_cast<unsigned>(a.seqs.batch)), dim3(128),
             4 * a.head_dim * sizeof(float), stream, a);
  return check_launch("attention_paged");
}

// Calls of the decode kernel (the others go to the tcgen05 kernel): up to 32 query rows
// per KV head, float32, and more heads per KV head than a tcgen05 tile has rows.
bool few_rows(dli_dtype dtype, int64_t group, int64_t max_new) {
  return dtype == DLI_DTYPE_F32 || group > 128 || group * max_new <= 32;
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
  if (batch > 65535) return fail(DLI_ERR_UNSUPPORTED, what + ": more than 65535 sequences");
  if (num_pages > INT_MAX || max_pages > (1ll << 30) / page_size)
    return fail(DLI_ERR_UNSUPPORTED, what + ": more than 2^30 rows per sequence or 2^31 pages");
  if (batch > 0 && (k_pages == nullptr || v_pages == nullptr || page_table == nullptr) && num_pages > 0 && max_pages > 0)
    return fail(DLI_ERR_INVALID_ARGUMENT, what + ": pages and page_table required");
  return DLI_OK;
}

dli_status check_rows(const std::string& what, int64_t tokens, int64_t batch, int64_t max_new, int64_t q_heads,
                      const void* positions, const void* starts) {
  if (tokens < 0 || max_new < 0 || q_heads <= 0) return fail(DLI_ERR_INVALID_ARGUMENT, what + ": bad sizes");
  if (positions == nullptr) return fail(DLI_ERR_INVALID_ARGUMENT, what + ": positions required");
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
  s.max_new = static_cast<int>(max_new);
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
  if (kv_dtype == DLI_DTYPE_FP4 && (!al || head_dim > 4096))
    return fail(DLI_ERR_INVALID_ARGUMENT, "qkv_rotary_paged: 4-bit pages need 16-byte aligned tensors and head_dim <= 4096");
  if (kv_dtype != DLI_DTYPE_FP4 && head_dim > 512)
    return fail(DLI_ERR_UNSUPPORTED, "qkv_rotary_paged: head_dim > 512");
  st = dispatch_float(dtype, what, [&](auto tag) {
    using T = decltype(tag);
    constexpr int V = Vec16<T>::N;
    if (kv_dtype == DLI_DTYPE_FP4) launch_append<T, Fp4, 16>(a, as_stream(stream));
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
  a.pages[0] = k_pages;
  a.pages[1] = v_pages;
  a.out[0] = k_out;
  a.out[1] = v_out;
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.hkv = static_cast<int>(kv_heads);
  a.head_dim = static_cast<int>(head_dim);
  a.count = count;
  const bool al = aligned(k_pages, 16) && aligned(v_pages, 16) && aligned(k_out, 16) && aligned(v_out, 16);
  if (kv_dtype == DLI_DTYPE_FP4 && !al)
    return fail(DLI_ERR_INVALID_ARGUMENT, "paged_gather: 4-bit pages need 16-byte aligned tensors");
  st = dispatch_float(dtype, what, [&](auto tag) {
    using T = decltype(tag);
    const bool vec = al && head_dim % 8 == 0;
    const int64_t items = count * (vec ? head_dim / 8 : head_dim);
    const int64_t walkers = std::min<int64_t>(ceil_div(items, 256),
                                              std::max<int64_t>(1, ceil_div(32ll * sm_count(), batch * kv_heads)));
    const dim3 grid(static_cast<unsigned>(walkers), static_cast<unsigned>(batch * kv_heads), 2u);
    if (kv_dtype == DLI_DTYPE_FP4) launch_pdl(paged_gather_kernel<T, Fp4, 8>, grid, dim3(256), 0, as_stream(stream), a);
    else if (vec) launch_pdl(paged_gather_kernel<T, T, 8>, grid, dim3(256), 0, as_stream(stream), a);
    else launch_pdl(paged_gather_kernel<T, T, 1>, grid, dim3(256), 0, as_stream(stream), a);
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
  const int64_t group = q_heads / kv_heads, max_keys = max_pages * page_size;
  (void)kv_dtype;
  if (few_rows(dtype, group, max_new)) return paged_decode_workspace(batch, kv_heads, group, max_new, head_dim, max_keys, dtype);
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
  a.softcap = softcap;
  a.v_scale = fp4 ? v_scale : 1.f;
  if (few_rows(dtype, a.group, max_new)) {
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
