// Shared pieces of the paged KV-cache kernels (append, gather, attention).
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace dli_sm100 {

// Element tag of 4-bit pages: E2M1 codes with one E4M3 scale per 16 elements.
struct Fp4 {};

// Arguments common to every kernel over pages. Row p of sequence b is row
// p & (page - 1) of page page_table[b * max_pages + (p >> page_shift)].
struct PagedSeqs {
  const int64_t* positions;  // rows cached before the call
  const int64_t* starts;     // packed row starts, or null: b * max_new
  const int32_t* page_table;
  int64_t tokens;
  int64_t num_pages, max_pages;
  int batch, max_new, page_shift;
  unsigned* err;
};

// The packed rows [row0, row0 + n) of sequence b and its cached rows before
// them. A sequence with starts or positions out of bounds has n = 0.
struct SeqRows {
  int64_t row0;
  int n, past;
};

__device__ __forceinline__ SeqRows seq_rows(const PagedSeqs& s, int b, bool report) {
  SeqRows r{0, 0, 0};
  const int64_t s0 = s.starts ? s.starts[b] : static_cast<int64_t>(b) * s.max_new;
  const int64_t s1 = s.starts ? s.starts[b + 1] : s0 + s.max_new;
  if (s0 < 0 || s1 < s0 || s1 > s.tokens || s1 - s0 > s.max_new) {
    if (report) set_device_error(s.err, kDevErrRaggedRows);
    return r;
  }
  const int64_t past = s.positions[b];
  if (past < 0 || past > (s.max_pages << s.page_shift) - (s1 - s0)) {
    if (report && s1 > s0) set_device_error(s.err, kDevErrKvCapacity);
    return r;
  }
  r.row0 = s0;
  r.n = static_cast<int>(s1 - s0);
  r.past = static_cast<int>(past);
  return r;
}

// Pool page of row p of sequence b (p inside the table), or -1 with the error
// word set when the table entry is outside the pool.
__device__ __forceinline__ int page_of(const PagedSeqs& s, int b, int p) {
  const int page = s.page_table[b * s.max_pages + (p >> s.page_shift)];
  if (page < 0 || page >= s.num_pages) {
    set_device_error(s.err, kDevErrPageIndex);
    return -1;
  }
  return page;
}

// Bytes of one (page, head) block.
__host__ __device__ constexpr int64_t fp4_block_bytes(int64_t page_rows, int64_t head_dim) {
  return page_rows * head_dim * 9 / 16;
}

// E4M3 byte -> float.
__device__ __forceinline__ float e4m3_value(unsigned byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}

// 2^-14 of an E2M1 nibble's value: its 3 magnitude bits as the low exponent bits and
// the top mantissa bit of a half (subnormals included).
__device__ __forceinline__ float e2m1_small(unsigned nibble) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(((nibble & 8u) << 12) | ((nibble & 7u) << 9))));
}
__device__ __forceinline__ float e2m1_value(unsigned nibble) { return e2m1_small(nibble) * 16384.f; }

// Element `c` of row `r` of a (page, head) block of 4-bit pages.
__device__ __forceinline__ float fp4_element(const uint8_t* block, int page_rows, int d, int r, int c) {
  const unsigned byte = block[static_cast<int64_t>(r) * (d / 2) + c / 2];
  const unsigned scale = block[static_cast<int64_t>(page_rows) * (d / 2) + static_cast<int64_t>(r) * (d / 16) + c / 16];
  return e2m1_value((c & 1) ? byte >> 4 : byte & 15u) * e4m3_value(scale);
}

// Dispatch of the attention over pages: every kernel takes these.
struct PagedAttnArgs {
  PagedSeqs seqs;
  const void* q;
  const void* k_pages;
  const void* v_pages;
  const float* slopes;  // per query head, or null
  void* out;
  int hq, hkv, group, head_dim;
  int window;         // keys visible to a row, its own included (INT_MAX: all)
  float scale;        // softmax scale, the cache's k_scale included
  float softcap;      // 0: none
  float v_scale;
};

}  // namespace dli_sm100
