// Attention of many new tokens over a paged KV cache on tcgen05 tensor cores:
// prompts and chunks of prompts, packed ragged batches, 16-bit or 4-bit pages, head
// dims 64 and 128, up to 128 query heads per KV head.
//
// A tile is 128 / group consecutive tokens of a sequence with all `group` query
// heads of one KV head (row = token * group + head; 126 of 128 rows at 7 heads),
// so a K/V block is fetched once for the whole group and a tile's rows differ by
// few tokens: few blocks are partly masked.
//
// One CTA = one tile, or one of `splits` shares of its key blocks when the tiles
// alone do not fill the GPU; 192 threads, two CTAs per SM:
//   warp 0     loads the Q tile once (a box of group x tokens of q by TMA), walks
//              the page table and loads 64-key K and V blocks (a box per page;
//              boxes past the sequence or of a bad page read as zeros) into rings
//              of 3 and 2 stages;
//   warp 1     allocates tensor memory and issues the MMAs, S_j = Q K_j^T and
//              O += P_j V_j, in the order S_0, S_1, P_0 V_0, S_2, ...;
//   warps 2-5  softmax, one thread per row: S from tensor memory, cap, bias and
//              mask, running maximum (moved only when it grows by more than 2^8,
//              so O is seldom rescaled) and sum in fp32, P as 16 bits over S's own
//              columns; at the end O / sum through shared memory to the rows, or
//              the share's (max, sum, O) to the workspace.
// 4-bit pages: no producer warp; four converter warps read codes and scales a
// block ahead into registers and write the K and V stages as halves (E2M1 x E4M3
// has 6 significant bits: exact), and the MMAs run in f16 for every model type. The
// softmax warps then write the Q tile, each row scaled by a power of two (exact), and
// undo the scale on the scores.
// Every wait is bounded; one that runs out sets the device error word.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "mma_sync.cuh"
#include "paged_attn.cuh"
#include "tcgen05.cuh"

namespace dli_sm100 {
namespace {

// warps: producer, MMA, 4 softmax; for 4-bit pages 4 softmax, 4 converters, MMA.
// The softmax warps hold a row of S: with converters in the CTA they take 32
// registers a thread from those (launched with 96: 128 x 128 + 128 x 64 + 32 x 96).
template <bool FP4>
struct Roles {
  static constexpr int kThreads = FP4 ? 288 : 192;
  static constexpr int kMma = FP4 ? 8 : 1;
  static constexpr int kSoftmax = FP4 ? 0 : 2;
  static constexpr int kConvert = 4;  // FP4 only
  static constexpr int kLaunchRegs = 96, kSoftmaxRegs = 128, kConvertRegs = 64;
  static_assert(128 * kSoftmaxRegs + 128 * kConvertRegs + 32 * kLaunchRegs <= 288 * kLaunchRegs, "register split");
};
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.f;  // log2: P <= 2^8 before O is rescaled
constexpr int BM = 128, BN = 64;

template <int D>
struct PrefillLayout {
  static constexpr int KST = 3, VST = 2;
  static constexpr int kBox = 128 * 128;
  static constexpr int kQBytes = (D / 64) * kBox;
  static constexpr int kKVBytes = (D / 64) * BN * 128;
  static constexpr int kKOff = kQBytes;
  static constexpr int kVOff = kKOff + KST * kKVBytes;
  static constexpr int kBarOff = kVOff + VST * kKVBytes;
  // q_full, k_full/empty, v_full/empty, s_full[2], s_empty[2], p_full, o_done, mma_done
  static constexpr int kBars = 1 + 2 * KST + 2 * VST + 4 + 3;
  static constexpr int kBytes = kBarOff + kBars * 8 + 16;  // two CTAs fit without alignment slack
  static constexpr uint32_t kTmemCols = 256;
  static constexpr uint32_t kOCol = 2 * BN;
  static_assert(kBytes <= 115712, "two CTAs per SM");
  static_assert(2 * BN + D <= 256, "tensor memory");
};

struct PrefillArgs {
  PagedAttnArgs a;
  int tile_tokens;  // 128 / group
  int splits;
  float* part_o;    // [units * splits][128][D]
  float2* part_ml;  // [units * splits][128]
  unsigned q_bytes; // of the Q box
};

// The shares of a tile's key blocks: at least 4 blocks each.
__device__ __forceinline__ int shares_of(int blocks, int splits) { return max(1, min(splits, blocks / 4)); }

struct Tile {
  SeqRows rows;
  int t0, tokens;       // of the tile
  int kv_len, key_lo;   // keys any of its rows sees: [key_lo, kv_len)
  int block0, blocks;
};

__device__ __forceinline__ Tile tile_of(const PrefillArgs& p, int b, int tile, bool report) {
  Tile x;
  x.rows = seq_rows(p.a.seqs, b, report);
  x.t0 = tile * p.tile_tokens;
  x.tokens = max(0, min(p.tile_tokens, x.rows.n - x.t0));
  const int pos0 = x.rows.past + x.t0;
  x.kv_len = pos0 + x.tokens;
  x.key_lo = p.a.window <= pos0 ? pos0 - p.a.window + 1 : 0;
  x.block0 = x.key_lo / BN;
  x.blocks = (x.kv_len + BN - 1) / BN - x.block0;
  return x;
}

__device__ __forceinline__ float max3f(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two fp32 lanes per instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{.reg .b64 ra, rb, rc, rd;\n\t"
      "mov.b64 ra, {%2, %3}; mov.b64 rb, {%4, %5}; mov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\t"
      "mov.b64 {%0, %1}, rd;}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3}; mov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\t"
      "mov.b64 {%0, %1}, rd;}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  const bool done = mbar_wait(bar, parity);
  return __all_sync(0xffffffffu, done && *abort_flag == 0);
}

// Halves of the codes in `w` (8 elements) times the scale pair `s`.
__device__ __forceinline__ uint4 fp4_halves(uint32_t w, uint32_t s) {
  return make_uint4(mul_half2(e2m1x2_to_half2<0>(w), s), mul_half2(e2m1x2_to_half2<1>(w), s),
                    mul_half2(e2m1x2_to_half2<2>(w), s), mul_half2(e2m1x2_to_half2<3>(w), s));
}

template <typename T, typename KV, int D>
__global__ void __launch_bounds__(Roles<std::is_same<KV, Fp4>::value>::kThreads, 2)
    attn_paged_prefill_kernel(const PrefillArgs p, const __grid_constant__ CUtensorMap tq,
                              const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv) {
  using L = PrefillLayout<D>;
  constexpr int KST = L::KST, VST = L::VST;
  constexpr bool kFp4 = std::is_same<KV, Fp4>::value;
  using MT = typename std::conditional<kFp4, __half, T>::type;  // MMA operand type
  using W = Roles<kFp4>;
  constexpr bool kBf16 = std::is_same<MT, __nv_bfloat16>::value;
  extern __shared__ uint8_t smem[];
  const PagedAttnArgs& a = p.a;
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) set_device_error(a.seqs.err, kDevErrAttentionTimeout);
    return;  // uniform for the CTA, nothing was started
  }
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + KST;
  uint64_t* v_full = k_empty + KST;
  uint64_t* v_empty = v_full + VST;
  uint64_t* s_full = v_empty + VST;
  uint64_t* s_empty = s_full + 2;
  uint64_t* p_full = s_empty + 2;
  uint64_t* o_done = p_full + 1;
  uint64_t* mma_done = o_done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_split = gridDim.x / p.splits;
  const int tile = per_split - 1 - static_cast<int>(blockIdx.x) / p.splits;  // the longest first
  const int share = static_cast<int>(blockIdx.x) % p.splits;
  const int kvh = blockIdx.y, b = blockIdx.z;

  // starts and positions may come from the kernel before
  pdl_wait();
  pdl_trigger();
  const Tile x = tile_of(p, b, tile, threadIdx.x == 0 && blockIdx.x == 0 && kvh == 0);
  if (x.tokens <= 0) return;  // uniform for the CTA, nothing was started
  const int shares = shares_of(x.blocks, p.splits);
  if (share >= shares) return;
  const int block_first = x.block0 + static_cast<int>(static_cast<int64_t>(share) * x.blocks / shares);
  const int nblocks = x.block0 + static_cast<int>(static_cast<int64_t>(share + 1) * x.blocks / shares) - block_first;
  // the last keys first: with a distance bias the maximum is then met early, and O is
  // not rescaled block after block
  auto key_of = [&](int j) { return (block_first + nblocks - 1 - j) * BN; };  // first key of step j

  if (threadIdx.x == 0) {
    constexpr int kWriters = kFp4 ? 4 : 1;  // warps that fill Q, K and V, or TMA
    mbar_init(q_full, kWriters);
    for (int s = 0; s < KST; ++s) {
      mbar_init(&k_full[s], kWriters);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < VST; ++s) {
      mbar_init(&v_full[s], kWriters);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_empty[s], 4);
    }
    mbar_init(p_full, 4);
    mbar_init(o_done, 1);
    mbar_init(mma_done, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == W::kMma) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int rows = x.tokens * a.group;  // of the 128
  const int pos0 = x.rows.past + x.t0;

  if (!kFp4 && warp == 0) {
    // ---- Q tile, then K and V blocks in the order the MMAs use them: K0, K1, V0, K2, V1, ...
    const int shift = a.seqs.page_shift, page_rows = 1 << shift;
    const int box_rows = min(page_rows, BN), boxes = BN / box_rows;
    const int32_t* ids = a.seqs.page_table + b * a.seqs.max_pages;
    const int last_page = (x.kv_len - 1) >> shift;
    const int none = static_cast<int>(a.seqs.num_pages);  // outside the map: reads as zeros
    if (lane == 0) {
      mbar_arrive_expect_tx(q_full, p.q_bytes);
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        tma_load_4d(smem + c * L::kBox, &tq, c * 64, kvh * a.group, static_cast<int>(x.rows.row0) + x.t0, 0, q_full);
    }
    auto page_for = [&](int j) {  // of lane's box of block j
      int page = none;
      const int i = j < nblocks ? (key_of(j) >> shift) + lane : 0;
      if (lane < boxes && j < nblocks && i <= last_page) {
        page = ids[i];
        if (page < 0 || page >= none) {
          set_device_error(a.seqs.err, kDevErrPageIndex);
          page = none;
        }
      }
      return page;
    };
    int k_issued = 0, v_issued = 0;
    bool ok = true;
    auto load = [&](int j, int page, bool is_k) {
      const int st = is_k ? j % KST : j % VST, round = is_k ? j / KST : j / VST;
      uint64_t* empty = is_k ? &k_empty[st] : &v_empty[st];
      uint64_t* full = is_k ? &k_full[st] : &v_full[st];
      const bool free_stage = mbar_wait(empty, (round & 1) ^ 1) && *abort_flag == 0;
      if (!__all_sync(0xffffffffu, free_stage)) return false;
      uint8_t* dst = smem + (is_k ? L::kKOff : L::kVOff) + st * L::kKVBytes;
      if (lane == 0) mbar_arrive_expect_tx(full, L::kKVBytes);
      __syncwarp();
      if (lane < boxes) {
        const int row = key_of(j) & (page_rows - 1);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(dst + c * (BN * 128) + lane * box_rows * 128, is_k ? &tk : &tv, c * 64, row, kvh, page, full);
      }
      __syncwarp();
      (is_k ? k_issued : v_issued) = j + 1;
      return true;
    };
    // the ids of the blocks ahead are asked for before they are needed
    int page0 = page_for(0), page1 = page_for(1), page2 = page_for(2);
    ok = load(0, page0, true);
    for (int j = 0; j < nblocks && ok; ++j) {
      const int page3 = page_for(j + 3);
      if (j + 1 < nblocks) ok = load(j + 1, page1, true);
      if (ok) ok = load(j, page0, false);
      page0 = page1;
      page1 = page2;
      page2 = page3;
    }
    if (!ok && lane == 0) {
      set_device_error(a.seqs.err, kDevErrAttentionTimeout);
      *abort_flag = 1;
    }
    // no copy may still be writing shared memory when the CTA exits
    mbar_wait(q_full, 0);
    for (int j = max(0, k_issued - KST); j < k_issued; ++j) mbar_wait(&k_full[j % KST], (j / KST) & 1);
    for (int j = max(0, v_issued - VST); j < v_issued; ++j) mbar_wait(&v_full[j % VST], (j / VST) & 1);
  } else if (warp == W::kMma) {
    if (lane == 0) {
      constexpr uint32_t idesc_s = umma_idesc_f16(kBf16, BM, BN);
      constexpr uint32_t idesc_o = umma_idesc_f16_bmn(kBf16, BM, D);
      const uint32_t q_addr = smem_u32(smem);
      auto qk = [&](int j) -> bool {
        const int s = j % KST, sb = j & 1;
        if (!mbar_wait(&k_full[s], (j / KST) & 1)) return false;
        if (!mbar_wait(&s_empty[sb], ((j >> 1) & 1) ^ 1) || *abort_flag) return false;
        tc_fence_after();
        const uint32_t k_addr = smem_u32(smem + L::kKOff + s * L::kKVBytes);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t ad = umma_desc_sw128(q_addr + (kk / 4) * L::kBox) + 2 * (kk % 4);
          const uint64_t bd = umma_desc_sw128(k_addr + (kk / 4) * (BN * 128)) + 2 * (kk % 4);
          umma_f16(tmem + static_cast<uint32_t>(sb * BN), ad, bd, idesc_s, kk > 0 ? 1u : 0u);
        }
        umma_commit(&k_empty[s]);
        umma_commit(&s_full[sb]);
        return true;
      };
      auto pv = [&](int j) -> bool {
        const int s = j % VST;
        if (!mbar_wait(p_full, j & 1)) return false;
        if (!mbar_wait(&v_full[s], (j / VST) & 1) || *abort_flag) return false;
        tc_fence_after();
        const uint32_t v_addr = smem_u32(smem + L::kVOff + s * L::kKVBytes);
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk) {
          // P_j over S_j's columns: S_{j+2}, issued later, cannot overwrite it before it is read
          const uint64_t bd = umma_desc_mn_sw128(v_addr + kk * 16 * 128, BN * 128, 1024);
          umma_f16_ts(tmem + L::kOCol, tmem + static_cast<uint32_t>((j & 1) * BN + kk * 8), bd, idesc_o,
                      (j > 0 || kk > 0) ? 1u : 0u);
        }
        umma_commit(&v_empty[s]);
        umma_commit(o_done);
        return true;
      };
      bool ok = mbar_wait(q_full, 0);
      if (ok) ok = qk(0);
      for (int j = 0; j < nblocks && ok; ++j) {
        if (j + 1 < nblocks) ok = qk(j + 1);
        if (ok) ok = pv(j);
      }
      if (!ok) {
        set_device_error(a.seqs.err, kDevErrAttentionTimeout);
        *abort_flag = 1;
      }
      // every issued MMA has finished before the CTA releases tensor memory
      umma_commit(mma_done);
      mbar_wait(mma_done, 0);
    }
  } else if (kFp4 && warp >= W::kConvert) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(W::kConvertRegs));
    // ---- converters: thread = half a key row; loads a block ahead, then K0, K1, V0, ...
    const int ct = threadIdx.x - W::kConvert * 32;
    const int key_row = ct & 63, half = ct >> 6;
    constexpr int WORDS = D / 16;  // code words of half a row
    constexpr int SB = D / 32;     // scale bytes
    const int shift = a.seqs.page_shift, page_rows = 1 << shift;
    const int32_t* ids = a.seqs.page_table + b * a.seqs.max_pages;
    const int64_t block_bytes = fp4_block_bytes(page_rows, D);
    const uint8_t* pages[2] = {static_cast<const uint8_t*>(a.k_pages), static_cast<const uint8_t*>(a.v_pages)};
    auto page_for = [&](int j) {
      const int key = j < nblocks ? key_of(j) + key_row : -1;
      if (key < 0 || key >= x.kv_len || key < x.key_lo) return -1;
      const int page = ids[key >> shift];
      if (page < 0 || page >= a.seqs.num_pages) {
        set_device_error(a.seqs.err, kDevErrPageIndex);
        return -1;
      }
      return page;
    };
    auto fetch = [&](int j, int page, int which, uint32_t (&w)[WORDS], uint32_t& sc) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[i] = 0u;
      sc = 0u;  // rows that are not of the tile's keys: zeros
      if (page < 0) return;
      const int r = (key_of(j) + key_row) & (page_rows - 1);
      const uint8_t* base = pages[which] + (static_cast<int64_t>(page) * a.hkv + kvh) * block_bytes;
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(base + r * (D / 2) + half * (D / 4) + i * 4);
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
      const uint8_t* s = base + page_rows * (D / 2) + r * (D / 16) + half * SB;
      sc = SB == 4 ? *reinterpret_cast<const uint32_t*>(s) : static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(s));
    };
    // the half row as swizzled 16-byte chunks of halves, then the warp's arrival
    auto put = [&](uint8_t* stage, const uint32_t (&w)[WORDS], uint32_t sc, uint64_t* full) {
      uint8_t* row = stage + (D == 128 ? half * (BN * 128) : 0) + key_row * 128;
      uint32_t s2 = 0u;
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        if (i % 4 == 0) s2 = e4m3x2_to_half2(sc >> (4 * i));
        const uint32_t s = i % 4 < 2 ? __byte_perm(s2, s2, 0x1010) : __byte_perm(s2, s2, 0x3232);
        const int ch = (D == 128 ? 0 : half * 4) + i;
        *reinterpret_cast<uint4*>(row + ((ch ^ (key_row & 7)) << 4)) = fp4_halves(w[i], s);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
    };
    uint32_t kw[WORDS], vw[WORDS], ks, vs;
    int page0 = page_for(0), page1 = page_for(1);
    fetch(0, page0, 0, kw, ks);
    fetch(0, page0, 1, vw, vs);
    bool ok = true;
    // V of block j is converted after K of block j + 1: the order of the MMAs
    for (int j = 0; j <= nblocks && ok; ++j) {
      const int page2 = page_for(j + 2);
      if (j < nblocks) {
        const int st = j % KST;
        ok = warp_wait(&k_empty[st], ((j / KST) & 1) ^ 1, abort_flag);
        if (!ok) break;
        put(smem + L::kKOff + st * L::kKVBytes, kw, ks, &k_full[st]);
        fetch(j + 1, page1, 0, kw, ks);
      }
      if (j > 0) {
        const int st = (j - 1) % VST;
        ok = warp_wait(&v_empty[st], (((j - 1) / VST) & 1) ^ 1, abort_flag);
        if (!ok) break;
        put(smem + L::kVOff + st * L::kKVBytes, vw, vs, &v_full[st]);
        fetch(j, page0, 1, vw, vs);
      }
      page0 = page1;
      page1 = page2;
    }
    if (!ok && lane == 0) {
      set_device_error(a.seqs.err, kDevErrAttentionTimeout);
      *abort_flag = 1;
    }
  } else {
    if constexpr (kFp4) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(W::kSoftmaxRegs));
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;  // tensor-memory lane = row of the tile
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const int tok = row / a.group, head = kvh * a.group + row - tok * a.group;
    const int pos = row < rows ? pos0 + tok : -1;  // rows past the tile compute what nobody reads
    const int lo = max(-1, pos - a.window);        // sees the keys in (lo, pos]
    const float slope = a.slopes && row < rows ? a.slopes[head] * kLog2e : 0.f;
    const bool cap = a.softcap > 0.f, bias = a.slopes != nullptr;
    const float cap_out = a.softcap * kLog2e;
    float in_scale = cap ? a.scale * 2.f * kLog2e / a.softcap : a.scale * kLog2e;
    if constexpr (kFp4) {
      // this thread's row of the Q tile, scaled by 2^-e with 2^e <= max|q| < 2^(e+1)
      const T* q = static_cast<const T*>(a.q) + ((x.rows.row0 + x.t0 + tok) * a.hq + head) * D;
      float big = 0.f;
      if (row < rows) {
#pragma unroll 4
        for (int c = 0; c < D; c += 8) {
          const Vec16<T> in = load16(q + c);
#pragma unroll
          for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(to_f32(in.e[i])));
        }
      }
      const int e = max(-120, min(120, static_cast<int>((__float_as_uint(big) >> 23) & 255u) - 127));
      const float down = __uint_as_float(static_cast<unsigned>(127 - e) << 23);
      in_scale *= __uint_as_float(static_cast<unsigned>(127 + e) << 23);
#pragma unroll 4
      for (int c = 0; c < D; c += 8) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (row < rows) {
          const Vec16<T> in = load16(q + c);
          v.x = pack16<MT>(to_f32(in.e[0]) * down, to_f32(in.e[1]) * down);
          v.y = pack16<MT>(to_f32(in.e[2]) * down, to_f32(in.e[3]) * down);
          v.z = pack16<MT>(to_f32(in.e[4]) * down, to_f32(in.e[5]) * down);
          v.w = pack16<MT>(to_f32(in.e[6]) * down, to_f32(in.e[7]) * down);
        }
        *reinterpret_cast<uint4*>(smem + (c >> 6) * L::kBox + row * 128 + ((((c >> 3) & 7) ^ (row & 7)) << 4)) = v;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    const float mul = cap || bias ? 1.f : in_scale;  // what the scores still want when the maximum is taken
    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < nblocks; ++j) {
      const int sb = j & 1;
      if (!warp_wait(&s_full[sb], (j >> 1) & 1, abort_flag)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float s[BN];
#pragma unroll
      for (int c = 0; c < BN / 32; ++c)
        tmem_ld_32x32b_x32(lane_base + static_cast<uint32_t>(sb * BN + c * 32), *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_empty[sb]);

      const int key0 = key_of(j);
      if (cap) {
#pragma unroll
        for (int i = 0; i < BN; ++i) s[i] = cap_out - 2.f * cap_out * rcp_approx(1.f + exp2_approx(s[i] * in_scale));
      }
      if (bias) {
        const float first = cap ? 1.f : in_scale, at = slope * static_cast<float>(key0 - pos);
#pragma unroll
        for (int i = 0; i < BN; i += 2) {
          const float2 far = fma2(make_float2(slope, slope), make_float2(i, i + 1), make_float2(at, at));
          const float2 y = fma2(make_float2(s[i], s[i + 1]), make_float2(first, first), far);
          s[i] = y.x;
          s[i + 1] = y.y;
        }
      }
      if (key0 + BN - 1 > pos0 || key0 <= pos0 + x.tokens - 1 - a.window) {
        const int end = pos - key0, begin = lo - key0;
#pragma unroll
        for (int i = 0; i < BN; ++i)
          if (i > end || i <= begin) s[i] = -INFINITY;
      }
      float mc[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) mc[k] = max3f(s[2 * k], s[2 * k + 1], -INFINITY);
#pragma unroll
      for (int i = 16; i < BN; i += 16)
#pragma unroll
        for (int k = 0; k < 8; ++k) mc[k] = max3f(mc[k], s[i + 2 * k], s[i + 2 * k + 1]);
      const float m_blk = max3f(max3f(mc[0], mc[1], mc[2]), max3f(mc[3], mc[4], mc[5]), fmaxf(mc[6], mc[7])) * mul;
      float alpha = 1.f;
      bool rescale_row = false;
      if (m_blk > m_used + kRescale) {  // from -inf: any visible key
        if (m_used != -INFINITY) {
          alpha = exp2_approx(m_used - m_blk);
          rescale_row = row < rows;
        }
        l *= alpha;
        m_used = m_blk;
      }
      if (__any_sync(0xffffffffu, rescale_row)) {
        // O holds P_0 V_0 + ... + P_{j-1} V_{j-1}: wait for the last of them. S_j's
        // commit covered P V_{j-2}, so o_done is at most one phase behind.
        if (!warp_wait(o_done, (j - 1) & 1, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(lane_base + L::kOCol + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
          tmem_st_32x32b_x32(lane_base + L::kOCol + c, r);
        }
        tmem_st_wait();
      }
      const float neg = m_used == -INFINITY ? 0.f : -m_used;
      uint32_t pk[BN / 2];
      float2 rs[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
      for (int i = 0; i < BN; i += 2) {
        float2 e = fma2(make_float2(s[i], s[i + 1]), make_float2(mul, mul), make_float2(neg, neg));
        e.x = exp2_approx(e.x);
        e.y = exp2_approx(e.y);
        rs[(i / 2) & 3] = add2(rs[(i / 2) & 3], e);
        pk[i / 2] = pack16<MT>(e.x, e.y);
      }
      const float2 sum = add2(add2(rs[0], rs[1]), add2(rs[2], rs[3]));
      l += sum.x + sum.y;
      // V rows that no row of the tile sees may hold anything: a zero weight must meet a zero
      const int z_end = x.kv_len - key0, z_begin = x.key_lo - key0;
      const bool stale = !kFp4 && (z_end < BN || z_begin > 0);  // the converters write zeros there
      if (stale) {
        if (!warp_wait(&v_full[j % VST], (j / VST) & 1, abort_flag)) {
          ok = false;
          break;
        }
        uint8_t* vt = smem + L::kVOff + (j % VST) * L::kKVBytes;
        for (int c = row; c < BN * (D / 8); c += BM) {
          const int box = c / (BN * 8), rem = c - box * (BN * 8);
          if (rem / 8 >= z_end || rem / 8 < z_begin)
            *reinterpret_cast<uint4*>(vt + box * BN * 128 + rem * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      tmem_st_32x32b_x32(lane_base + static_cast<uint32_t>(sb * BN), pk);
      tmem_st_wait();
      if (stale) fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    if (!ok && lane == 0) {
      set_device_error(a.seqs.err, kDevErrAttentionTimeout);
      *abort_flag = 1;
    }
    // every MMA has finished before O is read (o_done may be two phases behind here)
    bool have_o = ok;
    if (have_o && !warp_wait(mma_done, 0, abort_flag)) {
      if (lane == 0) set_device_error(a.seqs.err, kDevErrAttentionTimeout);
      have_o = false;
    }
    tc_fence_after();
    if (shares > 1) {
      // the share's O, unnormalised, its maximum and sum
      const int64_t unit = (static_cast<int64_t>(b) * a.hkv + kvh) * per_split + tile;
      const int64_t at = (unit * p.splits + share) * BM + row;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(lane_base + L::kOCol + c, r);
        tmem_ld_wait();
        if (row < rows && have_o) {
          float* dst = p.part_o + at * D + c;
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint4*>(dst + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
        }
      }
      if (row < rows) p.part_ml[at] = make_float2(have_o ? m_used : -INFINITY, l);
    } else {
      // O / l over the Q tile (the last Q K^T has completed), then whole head rows
      // of 16-byte chunks to the output
      const float inv = l > 0.f ? a.v_scale / l : 0.f;
      uint8_t* orow = smem + row * 128;
      const int r7 = row & 7;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(lane_base + L::kOCol + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          uint32_t v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[i] = have_o ? pack16<T>(__uint_as_float(r[q4 * 8 + 2 * i]) * inv, __uint_as_float(r[q4 * 8 + 2 * i + 1]) * inv) : 0u;
          const int ch = ((c & 63) >> 3) + q4;
          *reinterpret_cast<uint4*>(orow + (c >> 6) * L::kBox + ((ch ^ r7) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
      __syncwarp();
      // each warp stores its own 32 rows
      T* out = static_cast<T*>(a.out) + (x.rows.row0 + x.t0) * a.hq * D;
      constexpr int CPR = D / 8;
      const int r_end = min(32, rows - quarter * 32);
      for (int c = lane; c < r_end * CPR; c += 32) {
        const int r = quarter * 32 + c / CPR, ch = c % CPR;
        const int rt = r / a.group, rh = kvh * a.group + r - rt * a.group;
        const uint4 v = *reinterpret_cast<const uint4*>(smem + (ch >> 3) * L::kBox + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
        *reinterpret_cast<uint4*>(out + (static_cast<int64_t>(rt) * a.hq + rh) * D + ch * 8) = v;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == W::kMma) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

// Merges the shares of a tile in order.
template <typename T, int D>
__global__ void __launch_bounds__(256) attn_paged_prefill_combine_kernel(const PrefillArgs p) {
  DLI_PDL_ENTRY();
  const PagedAttnArgs& a = p.a;
  const int tile = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const Tile x = tile_of(p, b, tile, false);
  if (x.tokens <= 0) return;
  const int shares = shares_of(x.blocks, p.splits);
  if (shares == 1) return;
  const int64_t unit = (static_cast<int64_t>(b) * a.hkv + kvh) * gridDim.x + tile;
  const int rows = x.tokens * a.group;
  for (int c = threadIdx.x; c < rows * (D / 4); c += 256) {
    const int r = c / (D / 4), d = (c - r * (D / 4)) * 4;
    const int64_t at = unit * p.splits * BM + r;
    float top = -INFINITY, den = 0.f;
    for (int s = 0; s < shares; ++s) top = fmaxf(top, p.part_ml[at + s * BM].x);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < shares; ++s) {
      const float2 ml = p.part_ml[at + s * BM];
      if (ml.x == -INFINITY) continue;
      const float4 v = *reinterpret_cast<const float4*>(p.part_o + (at + s * BM) * D + d);
      const float f = exp2_approx(ml.x - top);
      den += ml.y * f;
      sum.x += v.x * f;
      sum.y += v.y * f;
      sum.z += v.z * f;
      sum.w += v.w * f;
    }
    const int tok = r / a.group, head = kvh * a.group + r - tok * a.group;
    const float inv = a.v_scale / den;
    uint2 v;
    v.x = pack16<T>(sum.x * inv, sum.y * inv);
    v.y = pack16<T>(sum.z * inv, sum.w * inv);
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + ((x.rows.row0 + x.t0 + tok) * a.hq + head) * D + d) = v;
  }
}

// ---- host ------------------------------------------------------------------------
struct PrefillPlan {
  int64_t tiles, units;
  int tile_tokens, splits;
  size_t part_o, workspace;
};

PrefillPlan plan_prefill(int64_t batch, int64_t hkv, int64_t group, int64_t max_new, int64_t head_dim, int64_t max_keys) {
  PrefillPlan p{};
  p.tile_tokens = static_cast<int>(BM / group);
  p.tiles = ceil_div(max_new, p.tile_tokens);
  p.units = p.tiles * hkv * batch;
  // as many shares of the keys as keep every CTA resident at once, at least 256 keys each
  const int64_t slots = 2ll * sm_count();
  p.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({slots / std::max<int64_t>(1, p.units), max_keys / (4 * BN), 64})));
  if (p.splits > 1) {
    p.part_o = static_cast<size_t>(p.units * p.splits * BM * head_dim) * 4;
    p.workspace = p.part_o + static_cast<size_t>(p.units * p.splits * BM) * 8;
  }
  return p;
}

template <typename T, typename KV, int D>
dli_status launch_prefill(const PagedAttnArgs& a, const PrefillPlan& plan, void* workspace, cudaStream_t stream) {
  using L = PrefillLayout<D>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr bool kFp4 = std::is_same<KV, Fp4>::value;
  CUtensorMap tq{}, tk{}, tv{};  // not used for 4-bit pages
  const int page_rows = 1 << a.seqs.page_shift;
  dli_status st = kFp4 ? DLI_OK : make_page_maps(a, kBf16 ? DLI_DTYPE_BF16 : DLI_DTYPE_F16, D, std::min(page_rows, BN), &tk, &tv);
  if (st != DLI_OK) return st;
  const uint64_t qd[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(a.hq), static_cast<uint64_t>(a.seqs.tokens), 1ull};
  const uint64_t row_bytes = static_cast<uint64_t>(a.hq) * D * 2;
  const uint64_t qs[3] = {static_cast<uint64_t>(D * 2), row_bytes, row_bytes * static_cast<uint64_t>(a.seqs.tokens)};
  const uint32_t qb[4] = {64u, static_cast<uint32_t>(a.group), static_cast<uint32_t>(plan.tile_tokens), 1u};
  if (!kFp4) st = make_map_4d(&tq, a.q, kBf16, qd, qs, qb);
  if (st != DLI_OK) return st;
  PrefillArgs p{};
  p.a = a;
  p.tile_tokens = plan.tile_tokens;
  p.splits = plan.splits;
  p.q_bytes = static_cast<unsigned>(plan.tile_tokens * a.group * D * 2);
  if (plan.splits > 1) {
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + plan.part_o);
  }
  auto kern = attn_paged_prefill_kernel<T, KV, D>;
  st = ensure_smem(reinterpret_cast<const void*>(kern), L::kBytes, "attention_paged");
  if (st != DLI_OK) return st;
  if (kFp4) {
    // the register split draws on what the CTA is launched with
    static const int regs = [&] {
      cudaFuncAttributes attr{};
      return cudaFuncGetAttributes(&attr, kern) == cudaSuccess ? attr.numRegs : 0;
    }();
    if (regs < Roles<true>::kLaunchRegs) return fail(DLI_ERR_UNSUPPORTED, "attention_paged: built with too few registers a thread");
  }
  const dim3 grid(static_cast<unsigned>(plan.tiles * plan.splits), static_cast<unsigned>(a.hkv),
                  static_cast<unsigned>(a.seqs.batch));
  launch_pdl(kern, grid, dim3(Roles<kFp4>::kThreads), L::kBytes, stream, p, tq, tk, tv);
  if (plan.splits > 1)
    launch_pdl(attn_paged_prefill_combine_kernel<T, D>,
               dim3(static_cast<unsigned>(plan.tiles), static_cast<unsigned>(a.hkv), static_cast<unsigned>(a.seqs.batch)),
               dim3(256), 0, stream, p);
  return check_launch("attention_paged", plan.splits > 1 ? 2 : 1);
}

int64_t keys_of(const PagedAttnArgs& a) {
  return std::min<int64_t>(a.seqs.max_pages << a.seqs.page_shift, static_cast<int64_t>(a.window) + a.seqs.max_new);
}

}  // namespace

bool paged_prefill_serves(const PagedAttnArgs& a, dli_dtype dtype, dli_dtype kv_dtype) {
  if ((dtype != DLI_DTYPE_BF16 && dtype != DLI_DTYPE_F16) || (kv_dtype != dtype && kv_dtype != DLI_DTYPE_FP4)) return false;
  if (a.head_dim != 64 && a.head_dim != 128) return false;
  if (a.group > BM || a.hkv > 65535 || a.seqs.num_pages < 1 || a.seqs.tokens > INT_MAX) return false;
  for (const void* p : {a.q, a.k_pages, a.v_pages, static_cast<const void*>(a.out)})
    if (!aligned(p, 16)) return false;
  return true;
}

size_t paged_prefill_workspace(int64_t batch, int64_t hkv, int64_t group, int64_t max_new, int64_t head_dim, int64_t max_keys) {
  return plan_prefill(batch, hkv, group, max_new, head_dim, max_keys).workspace;
}

dli_status run_paged_prefill(const PagedAttnArgs& a, dli_dtype dtype, dli_dtype kv_dtype, void* workspace,
                             size_t workspace_bytes, cudaStream_t stream) {
  const PrefillPlan plan = plan_prefill(a.seqs.batch, a.hkv, a.group, a.seqs.max_new, a.head_dim, keys_of(a));
  if (plan.workspace > 0 && (workspace == nullptr || workspace_bytes < plan.workspace || !aligned(workspace, 16)))
    return fail(DLI_ERR_WORKSPACE, "attention_paged: a 16-byte aligned workspace of " + std::to_string(plan.workspace) + " bytes is needed");
  if (kv_dtype == DLI_DTYPE_FP4) {
    if (dtype == DLI_DTYPE_BF16)
      return a.head_dim == 64 ? launch_prefill<__nv_bfloat16, Fp4, 64>(a, plan, workspace, stream)
                              : launch_prefill<__nv_bfloat16, Fp4, 128>(a, plan, workspace, stream);
    return a.head_dim == 64 ? launch_prefill<__half, Fp4, 64>(a, plan, workspace, stream)
                            : launch_prefill<__half, Fp4, 128>(a, plan, workspace, stream);
  }
  if (dtype == DLI_DTYPE_BF16)
    return a.head_dim == 64 ? launch_prefill<__nv_bfloat16, __nv_bfloat16, 64>(a, plan, workspace, stream)
                            : launch_prefill<__nv_bfloat16, __nv_bfloat16, 128>(a, plan, workspace, stream);
  return a.head_dim == 64 ? launch_prefill<__half, __half, 64>(a, plan, workspace, stream)
                          : launch_prefill<__half, __half, 128>(a, plan, workspace, stream);
}

}  // namespace dli_sm100
