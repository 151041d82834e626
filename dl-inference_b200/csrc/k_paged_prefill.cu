// Attention of many new tokens over a paged KV cache on tcgen05 tensor cores:
// prompts and chunks of prompts, packed ragged batches, 16-bit or 4-bit pages, head
// dims 64 and 128, up to 128 query heads per KV head.
//
// A tile is 128 / group consecutive tokens of a sequence with all `group` query
// heads of one KV head (row = token * group + head; 126 of 128 rows at 7 heads),
// so a K/V block is fetched once for the whole group and a tile's rows differ by
// few tokens: few blocks are partly masked.
//
// Many tiles: the grid is their list, by groups of (sequence, KV head) pairs whose K/V
// stay in L2, in a group the sequences' tiles by their index up to max_new, from the last
// (the longest first where the sequences have as many cached rows; a single token is tile 0
// and comes last, however long its cache). A CTA that works claims the next one of the list
// from the hardware scheduler (cluster launch control) while it computes, so two CTAs
// per SM stay for the whole call, one tile's end overlaps the next one's start, and a
// ragged batch is balanced as it runs (which CTA computes a tile changes nothing in it).
// Prompts beside single tokens suit neither rule: 1 x 2048 tokens 44 us, 31 x 1 over 8,000
// to 32,000 keys 196 in the decode kernel, both in one call, here, 612.
// Few tiles: each tile's keys are split evenly into parts, which are items of the list
// like tiles; they store their (max, sum, O) in the workspace, and a second kernel merges
// them in order.
// 192 threads:
//   warp 0     loads each Q tile (a box of group x tokens of q by TMA), walks the page
//              table and loads 64-key K and V blocks (a box per page; boxes past the
//              sequence or of a bad page read as zeros) into rings of 3 and 2 stages,
//              running ahead into the next tile;
//   warp 1     allocates tensor memory and issues the MMAs, S_j = Q K_j^T and
//              O += P_j V_j, in the order S_0, S_1, P_0 V_0, S_2, ...;
//   warps 2-5  softmax, one thread per row: S from tensor memory, cap, bias and
//              mask, running maximum (moved only when it grows by more than 2^8,
//              so O is seldom rescaled) and sum in fp32, P as 16 bits over S's own
//              columns; at the end O / sum to the rows, or the part's (max, sum, O)
//              to the workspace, while the next tile's first S is computed.
// 4-bit pages: no producer warp; four converter warps read codes and scales a
// block ahead into registers and write the K and V stages as halves (E2M1 x E4M3
// has 6 significant bits: exact), and the MMAs run in f16 for every model type. The
// softmax warps then write the Q tile, each row scaled by a power of two so that its
// largest element is in [1, 2) (halves keep smaller ones to 2^-25 of it), and undo the
// scale on the scores.
// P is rounded to the model's 16-bit type for P V (to halves over 4-bit pages); sums and O
// stay in fp32. Against 64 bits a bf16 output is off by 2.1e-3, where its own rounding
// gives 1.6e-3, f16 2.4e-4 and 2.1e-4.
// Every wait is bounded; one that runs out sets the device error word and winds the
// CTA down.
//
// Bound by the chain S -> softmax -> P V -> next S of each CTA (tensor pipe busy 38% of the
// active cycles, MUFU 39%, issue 39%, L2 25%; two threads per row, 96 registers each, 402 us
// instead of 365): 16 prompts of up to 2048 tokens, 28/4 heads of 128, bf16: 365 us = 787
// TFLOP/s in a graph of 12 calls, 416 = 693 called one by one for seconds, at the clocks of
// the power cap (466 when a grid of whole tiles had no claiming; 64 keys a block keep two CTAs in an
// SM's tensor memory). 2 chunks of up to 383 tokens over 8000 keys, window 4096, bias, 16
// heads of 64: 39 us (issue 39%, MUFU 34%, tensor 17% busy). 4-bit pages, 4 chunks of up
// to 301 tokens over 3001 keys, 28/4 heads: 83 us (issue 43%, ALU 35%, tensor 26% busy, the
// converters' loads), over 16-bit pages 65.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "mma_sync.cuh"
#include "paged_attn.cuh"
#include "tcgen05.cuh"

namespace dli_sm100 {
namespace {

// warps: producer, MMA, 4 softmax; for 4-bit pages 4 softmax, 4 converters, MMA,
// scheduler. The softmax warps hold a row of S: with converters in the CTA they take 32
// registers a thread from those (launched with 96: 128 x 128 + 128 x 64 + 64 x 96).
template <bool FP4>
struct Roles {
  static constexpr int kThreads = FP4 ? 320 : 192;
  static constexpr int kMma = FP4 ? 8 : 1;
  static constexpr int kSoftmax = FP4 ? 0 : 2;
  static constexpr int kConvert = 4, kSchedule = 9;  // FP4 only
  static constexpr int kLaunchRegs = 96, kSoftmaxRegs = 128, kConvertRegs = 64;
  static_assert(128 * kSoftmaxRegs + 128 * kConvertRegs + 64 * kLaunchRegs <= 320 * kLaunchRegs, "register split");
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
  static constexpr int kTiles = 16 + 2 * 48;  // the hardware scheduler's answer, two tiles; then the barriers:
  // q_full, q_empty, k_full/empty, v_full/empty, s_full[2], p_full[2], o_done,
  // o_full, o_empty, mma_done, claimed, near_end, tile_full[2], tile_empty[2]
  static constexpr int kBars = 2 + 2 * KST + 2 * VST + 4 + 4 + 6;
  static constexpr int kBytes = kBarOff + kTiles + kBars * 8 + 16;  // two CTAs fit without alignment slack
  static constexpr uint32_t kTmemCols = 256;
  static constexpr uint32_t kOCol = 2 * BN;
  static_assert(kBytes <= 115712, "two CTAs per SM");
  static_assert(2 * BN + D <= 256, "tensor memory");
};

struct PrefillArgs {
  PagedAttnArgs a;
  int tile_tokens;  // 128 / group
  int tiles;        // of a sequence of max_new tokens
  int split;        // parts of a tile's keys, at most
  int min_part;     // key blocks of a part, at least
  int pairs_group;  // (sequence, KV head) pairs whose tiles are interleaved
  int wide_out;     // out is 32-byte aligned
  float* part_o;    // [tiles x split][D / 4][128][4]
  float2* part_ml;  // [tiles x split][128]
  unsigned q_bytes; // of the Q box
};

// A tile, or the part of one at hand; 48 bytes, as it lies in shared memory.
struct alignas(16) Tile {
  int b, kvh, row0, past;
  int t0, tokens;            // of the tile
  int kv_len, key_lo;        // keys any of its rows sees: [key_lo, kv_len)
  int block_first, nblocks;  // of the part; no blocks: the end
  int slot;                  // of the part in the workspace, -1: the whole tile
  int unused;
  // the last keys first: with a distance bias the maximum is then met early, and O is
  // not rescaled block after block
  __device__ __forceinline__ int key_of(int j) const { return (block_first + nblocks - 1 - j) * BN; }
};
static_assert(sizeof(Tile) == 48, "three 16-byte words");

// Sets x to all of tile `tile` of sequence b; false when it has no tokens.
__device__ __forceinline__ bool tile_set(const PrefillArgs& p, const SeqRows& rows, int b, int kvh, int tile, Tile& x) {
  x.b = b;
  x.kvh = kvh;
  x.row0 = static_cast<int>(rows.row0);
  x.past = rows.past;
  x.t0 = tile * p.tile_tokens;
  x.tokens = min(p.tile_tokens, rows.n - x.t0);
  if (x.tokens <= 0) return false;
  const int pos0 = x.past + x.t0;
  x.kv_len = pos0 + x.tokens;
  x.key_lo = p.a.window <= pos0 ? pos0 - p.a.window + 1 : 0;
  x.block_first = x.key_lo / BN;
  x.nblocks = (x.kv_len + BN - 1) / BN - x.block_first;
  x.slot = -1;
  return true;
}
// The parts of a tile with `blocks` blocks, by its sequence's length.
__device__ __forceinline__ int parts_of(const PrefillArgs& p, int blocks) { return max(1, min(p.split, blocks / p.min_part)); }

// The one warp that finds the CTA's next item: its own of the grid, then what the
// hardware scheduler grants.
struct Scheduler {
  const PrefillArgs& p;
  uint8_t* answer;
  uint64_t* claimed;
  int lane;
  int claims = 0;  // answered
  bool begun = false, open = false;

  // Item `at` of the grid's list; false when there is nothing to do in it. Order: parts,
  // groups of pairs, tiles from the last that max_new allows, the pairs of the group.
  __device__ __forceinline__ bool item(int at, Tile& x) {
    const int pairs = p.a.hkv * p.a.seqs.batch, units = pairs * p.tiles;
    const int part = at / units, unit = at - part * units;
    const int group = unit / p.tiles / p.pairs_group;
    const int first = group * p.pairs_group, size = min(p.pairs_group, pairs - first);
    const int in_group = unit - first * p.tiles;
    const int rank = in_group / size, pair = first + in_group - rank * size;
    const int seq = pair / p.a.hkv, tile = p.tiles - 1 - rank;
    const SeqRows rows = seq_rows(p.a.seqs, seq, lane == 0 && tile == 0);
    if (!tile_set(p, rows, seq, pair - seq * p.a.hkv, tile, x)) return false;
    const int parts = parts_of(p, x.nblocks);
    if (part >= parts) return false;
    if (parts > 1) {
      const int64_t blocks = x.nblocks;
      const int lo = static_cast<int>(part * blocks / parts);
      x.nblocks = static_cast<int>((part + 1) * blocks / parts) - lo;
      x.block_first += lo;
      x.slot = (pair * p.tiles + tile) * p.split + part;
    }
    return true;
  }
  // Asks for another item: a few key blocks before a tile's end (not earlier: what is
  // claimed waits for this CTA, while another may be idle).
  __device__ __forceinline__ void ask() {
    if (lane == 0) {
      mbar_arrive_expect_tx(claimed, 16);
      claim_next_cta(answer, claimed);
    }
    open = true;
  }
  __device__ bool next(Tile& x, bool& ok) {
    while (true) {
      int at = static_cast<int>(blockIdx.x);
      if (begun) {
        if (!__all_sync(0xffffffffu, mbar_wait(claimed, claims & 1))) {
          ok = false;
          return false;
        }
        at = claimed_cta(answer);
        open = false;
        ++claims;
        fence_proxy_async_smem();  // read before it is written again
        __syncwarp();
        if (at < 0) return false;
      }
      begun = true;
      if (item(at, x)) return true;
      ask();
    }
  }
};

// The tiles as the scheduling warp passes them to the others, through two slots. It may
// look through very many items without a tile first (2.4 ns each, over all CTAs: 2^30 of
// them 2.5 s, more than one wait lasts).
struct TileQueue {
  static constexpr int kPatience = 8;  // waits
  uint8_t* slots;
  uint64_t* full;
  uint64_t* empty;
  int n = 0;
  // By the scheduling warp; x.nblocks = 0 at the end.
  __device__ __forceinline__ bool put(const Tile& x, int lane) {
    const bool free_slot = mbar_wait(&empty[n & 1], ((n >> 1) & 1) ^ 1);
    if (!__all_sync(0xffffffffu, free_slot)) return false;
    if (lane == 0) {
      const uint4* from = reinterpret_cast<const uint4*>(&x);
      uint4* to = reinterpret_cast<uint4*>(slots + 48 * (n & 1));
      to[0] = from[0];
      to[1] = from[1];
      to[2] = from[2];
      mbar_arrive(&full[n & 1]);
    }
    __syncwarp();
    ++n;
    return true;
  }
  // By another warp, or by one thread of it (single). False at the end, and with ok
  // false when the wait ran out.
  __device__ __forceinline__ bool get(Tile& x, bool single, volatile int* abort_flag, bool& ok) {
    bool got = false;
    for (int tries = 0; !got && tries < kPatience && *abort_flag == 0; ++tries) got = mbar_wait(&full[n & 1], (n >> 1) & 1);
    got = got && *abort_flag == 0;
    if (!single) got = __all_sync(0xffffffffu, got);
    if (!got) {
      ok = false;
      return false;
    }
    const uint4* from = reinterpret_cast<const uint4*>(slots + 48 * (n & 1));
    uint4* to = reinterpret_cast<uint4*>(&x);
    to[0] = from[0];
    to[1] = from[1];
    to[2] = from[2];
    if (!single) __syncwarp();
    if (single || (threadIdx.x & 31) == 0) mbar_arrive(&empty[n & 1]);
    ++n;
    return x.nblocks > 0;
  }
};

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

// Two of capped_score's small ones, by the same roundings.
__device__ __forceinline__ float2 capped_small(float2 z, float cap2) {
  auto both = [](float x) { return make_float2(x, x); };
  const float2 s = make_float2(z.x * z.x, z.y * z.y);
  float2 t = fma2(s, both(kTanh4), both(kTanh3));
  t = fma2(s, t, both(kTanh2));
  t = fma2(s, t, both(kTanh1));
  t = fma2(s, t, both(1.f));
  const float first = kTanh0 * cap2;
  return make_float2(t.x * (z.x * first), t.y * (z.y * first));
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
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::kBarOff + L::kTiles);
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_empty + 1;
  uint64_t* k_empty = k_full + KST;
  uint64_t* v_full = k_empty + KST;
  uint64_t* v_empty = v_full + VST;
  uint64_t* s_full = v_empty + VST;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_done = p_full + 2;
  uint64_t* o_full = o_done + 1;
  uint64_t* o_empty = o_full + 1;
  uint64_t* mma_done = o_empty + 1;
  uint64_t* claimed = mma_done + 1;
  uint64_t* near_end = claimed + 1;
  uint64_t* tile_full = near_end + 1;
  uint64_t* tile_empty = tile_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tile_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    constexpr int kWriters = kFp4 ? 4 : 1;  // warps that fill Q, K and V, or TMA
    mbar_init(q_full, kWriters);
    mbar_init(q_empty, 1);
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
      mbar_init(&p_full[s], 4);
    }
    mbar_init(o_done, 1);
    mbar_init(o_full, 1);
    mbar_init(o_empty, 4);
    mbar_init(mma_done, 1);
    mbar_init(claimed, 1);
    mbar_init(near_end, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&tile_full[s], 1);
      mbar_init(&tile_empty[s], kFp4 ? 9 : 5);  // the MMA thread, softmax warps, converters
    }
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
  pdl_wait();
  pdl_trigger();
  TileQueue tiles{smem + L::kBarOff + 16, tile_full, tile_empty};
  Tile x;
  bool ok = true;
  int g0 = 0;    // key blocks of the tiles before this one: stages and phases run on
  int tile_n = 0;  // tiles before this one

  if (!kFp4 && warp == 0) {
    // ---- Q tiles, and K and V blocks in the order the MMAs use them: K0, K1, V0, K2, V1, ...
    const int shift = a.seqs.page_shift, page_rows = 1 << shift;
    const int box_rows = min(page_rows, BN), boxes = BN / box_rows;
    const int none = static_cast<int>(a.seqs.num_pages);  // outside the map: reads as zeros
    int k_issued = 0, v_issued = 0, q_issued = 0;
    Scheduler scheduler{p, smem + L::kBarOff, claimed, lane};
    while (ok) {
      if (!scheduler.next(x, ok)) x.nblocks = 0;
      ok = tiles.put(x, lane) && ok;
      if (!ok || x.nblocks == 0) break;
      const int32_t* ids = a.seqs.page_table + x.b * a.seqs.max_pages;
      const int first_page = x.key_lo >> shift, last_page = (x.kv_len - 1) >> shift;  // others may be gone
      auto page_for = [&](int j) {  // of lane's box of step j
        int page = none;
        const int i = j < x.nblocks ? (x.key_of(j) >> shift) + lane : 0;
        if (lane < boxes && j < x.nblocks && i >= first_page && i <= last_page) {
          page = ids[i];
          if (page < 0 || page >= none) {
            set_device_error(a.seqs.err, kDevErrPageIndex);
            page = none;
          }
        }
        return page;
      };
      auto load = [&](int j, int page, bool is_k) {
        const int g = g0 + j;
        const int st = is_k ? g % KST : g % VST, round = is_k ? g / KST : g / VST;
        uint64_t* empty = is_k ? &k_empty[st] : &v_empty[st];
        uint64_t* full = is_k ? &k_full[st] : &v_full[st];
        const bool free_stage = mbar_wait(empty, (round & 1) ^ 1) && *abort_flag == 0;
        if (!__all_sync(0xffffffffu, free_stage)) return false;
        uint8_t* dst = smem + (is_k ? L::kKOff : L::kVOff) + st * L::kKVBytes;
        if (lane == 0) mbar_arrive_expect_tx(full, L::kKVBytes);
        __syncwarp();
        if (lane < boxes) {
          const int row = x.key_of(j) & (page_rows - 1);
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_load_4d(dst + c * (BN * 128) + lane * box_rows * 128, is_k ? &tk : &tv, c * 64, row, x.kvh, page, full);
        }
        __syncwarp();
        (is_k ? k_issued : v_issued) = g + 1;
        return true;
      };
      // the ids of the steps ahead are asked for before they are needed
      int page0 = page_for(0), page1 = page_for(1), page2 = page_for(2);
      // K of the first step does not wait for the Q tile's buffer
      ok = load(0, page0, true);
      if (!ok) break;
      const bool q_free = mbar_wait(q_empty, (tile_n & 1) ^ 1) && *abort_flag == 0;
      ok = __all_sync(0xffffffffu, q_free);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(q_full, p.q_bytes);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(smem + c * L::kBox, &tq, c * 64, x.kvh * a.group, x.row0 + x.t0, 0, q_full);
      }
      __syncwarp();
      q_issued = tile_n + 1;
      for (int j = 0; j < x.nblocks && ok; ++j) {
        if (j == max(0, x.nblocks - 2)) scheduler.ask();
        const int page3 = page_for(j + 3);
        if (j + 1 < x.nblocks) ok = load(j + 1, page1, true);
        if (ok) ok = load(j, page0, false);
        page0 = page1;
        page1 = page2;
        page2 = page3;
      }
      g0 += x.nblocks;
      ++tile_n;
    }
    if (!ok && lane == 0) {
      set_device_error(a.seqs.err, kDevErrAttentionTimeout);
      *abort_flag = 1;
    }
    // no copy may still be writing shared memory when the CTA exits
    if (scheduler.open) mbar_wait(claimed, scheduler.claims & 1);
    if (q_issued > 0) mbar_wait(q_full, (q_issued - 1) & 1);
    for (int g = max(0, k_issued - KST); g < k_issued; ++g) mbar_wait(&k_full[g % KST], (g / KST) & 1);
    for (int g = max(0, v_issued - VST); g < v_issued; ++g) mbar_wait(&v_full[g % VST], (g / VST) & 1);
  } else if (warp == W::kMma) {
    if (lane == 0) {
      constexpr uint32_t idesc_s = umma_idesc_f16(kBf16, BM, BN);
      constexpr uint32_t idesc_o = umma_idesc_f16_bmn(kBf16, BM, D);
      const uint32_t q_addr = smem_u32(smem);
      while (ok && tiles.get(x, true, abort_flag, ok)) {
        auto qk = [&](int j) -> bool {
          const int g = g0 + j, s = g % KST, sb = g & 1;
          if (!mbar_wait(&k_full[s], (g / KST) & 1)) return false;
          // S_g's buffer held S and P_{g-2}, whose P V is issued: no wait for the readers
          if (*abort_flag) return false;
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
          if (j == x.nblocks - 1) umma_commit(q_empty);
          return true;
        };
        auto pv = [&](int j) -> bool {
          const int g = g0 + j, s = g % VST;
          if (!mbar_wait(&p_full[g & 1], (g >> 1) & 1)) return false;
          if (!mbar_wait(&v_full[s], (g / VST) & 1) || *abort_flag) return false;
          // O of the tile before has been read
          if (j == 0 && tile_n > 0 && !mbar_wait(o_empty, (tile_n - 1) & 1)) return false;
          tc_fence_after();
          const uint32_t v_addr = smem_u32(smem + L::kVOff + s * L::kKVBytes);
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk) {
            // P_j over S_j's columns: S_{j+2}, issued later, cannot overwrite it before it is read
            const uint64_t bd = umma_desc_mn_sw128(v_addr + kk * 16 * 128, BN * 128, 1024);
            umma_f16_ts(tmem + L::kOCol, tmem + static_cast<uint32_t>((g & 1) * BN + kk * 8), bd, idesc_o,
                        (j > 0 || kk > 0) ? 1u : 0u);
          }
          umma_commit(&v_empty[s]);
          umma_commit(o_done);
          if (j == x.nblocks - 1) umma_commit(o_full);
          return true;
        };
        ok = mbar_wait(q_full, tile_n & 1);
        if (ok) ok = qk(0);
        for (int j = 0; j < x.nblocks && ok; ++j) {
          if (j + 1 < x.nblocks) ok = qk(j + 1);
          if (ok) ok = pv(j);
        }
        g0 += x.nblocks;
        ++tile_n;
      }
      if (!ok) {
        set_device_error(a.seqs.err, kDevErrAttentionTimeout);
        *abort_flag = 1;
      }
      // every issued MMA has finished before the CTA releases tensor memory
      umma_commit(mma_done);
      mbar_wait(mma_done, 0);
    }
  } else if (kFp4 && warp == W::kSchedule) {
    Scheduler scheduler{p, smem + L::kBarOff, claimed, lane};
    while (ok) {
      if (!scheduler.next(x, ok)) x.nblocks = 0;
      ok = tiles.put(x, lane) && ok;
      if (!ok || x.nblocks == 0) break;
      // a whole tile may take longer than one wait lasts: as long as its blocks may take
      bool near = false;
      for (int tries = 0; !near && tries <= x.nblocks && *abort_flag == 0; ++tries) near = mbar_wait(near_end, tile_n & 1);
      ok = __all_sync(0xffffffffu, near);
      if (!ok) break;
      scheduler.ask();
      ++tile_n;
    }
    if (!ok && lane == 0) {
      set_device_error(a.seqs.err, kDevErrAttentionTimeout);
      *abort_flag = 1;
    }
    if (scheduler.open) mbar_wait(claimed, scheduler.claims & 1);  // no answer is still to be written
  } else if (kFp4 && warp >= W::kConvert) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(W::kConvertRegs));
    // ---- converters: thread = half a key row; loads a block ahead, then K0, K1, V0, ...
    const int ct = threadIdx.x - W::kConvert * 32;
    const int key_row = ct & 63, half = ct >> 6;
    constexpr int WORDS = D / 16;  // code words of half a row
    constexpr int SB = D / 32;     // scale bytes
    const int shift = a.seqs.page_shift, page_rows = 1 << shift;
    const int64_t block_bytes = fp4_block_bytes(page_rows, D);
    const uint8_t* pages[2] = {static_cast<const uint8_t*>(a.k_pages), static_cast<const uint8_t*>(a.v_pages)};
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
    while (ok && tiles.get(x, false, abort_flag, ok)) {
      const int32_t* ids = a.seqs.page_table + x.b * a.seqs.max_pages;
      auto page_for = [&](int j) {
        const int key = j < x.nblocks ? x.key_of(j) + key_row : -1;
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
        const int r = (x.key_of(j) + key_row) & (page_rows - 1);
        const uint8_t* base = pages[which] + (static_cast<int64_t>(page) * a.hkv + x.kvh) * block_bytes;
#pragma unroll
        for (int i = 0; i < WORDS; i += 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(base + r * (D / 2) + half * (D / 4) + i * 4);
          w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
        }
        const uint8_t* s = base + page_rows * (D / 2) + r * (D / 16) + half * SB;
        sc = SB == 4 ? *reinterpret_cast<const uint32_t*>(s) : static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(s));
      };
      uint32_t kw[WORDS], vw[WORDS], ks, vs;
      int page0 = page_for(0), page1 = page_for(1);
      fetch(0, page0, 0, kw, ks);
      fetch(0, page0, 1, vw, vs);
      // V of step j is converted after K of step j + 1: the order of the MMAs
      for (int j = 0; j <= x.nblocks; ++j) {
        const int page2 = page_for(j + 2);
        if (ct == 0 && j == max(0, x.nblocks - 2)) mbar_arrive(near_end);
        if (j < x.nblocks) {
          const int g = g0 + j, st = g % KST;
          ok = warp_wait(&k_empty[st], ((g / KST) & 1) ^ 1, abort_flag);
          if (!ok) break;
          put(smem + L::kKOff + st * L::kKVBytes, kw, ks, &k_full[st]);
          fetch(j + 1, page1, 0, kw, ks);
        }
        if (j > 0) {
          const int g = g0 + j - 1, st = g % VST;
          ok = warp_wait(&v_empty[st], ((g / VST) & 1) ^ 1, abort_flag);
          if (!ok) break;
          put(smem + L::kVOff + st * L::kKVBytes, vw, vs, &v_full[st]);
          fetch(j, page0, 1, vw, vs);
        }
        page0 = page1;
        page1 = page2;
      }
      g0 += x.nblocks;
      ++tile_n;
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
    const int tok = row / a.group, in_group = row - tok * a.group;
    const bool cap = a.softcap > 0.f, bias = a.slopes != nullptr;
    const float cap2 = 2.f * a.softcap * kLog2e;
    while (ok && tiles.get(x, false, abort_flag, ok)) {
      const int rows = x.tokens * a.group;  // of the 128
      const int pos0 = x.past + x.t0;
      const int head = x.kvh * a.group + in_group;
      const int pos = row < rows ? pos0 + tok : -1;  // rows past the tile compute what nobody reads
      const int lo = max(-1, pos - a.window);        // sees the keys in (lo, pos]
      const float slope = bias && row < rows ? a.slopes[head] * kLog2e : 0.f;
      float in_scale = cap ? a.scale * 2.f * kLog2e / a.softcap : a.scale * kLog2e;
      if constexpr (kFp4) {
        // this thread's row of the Q tile (every S of the tile before has been read, so
        // its Q has too), scaled by 2^-e with 2^e <= max|q| < 2^(e+1)
        const T* q = static_cast<const T*>(a.q) + (static_cast<int64_t>(x.row0 + x.t0 + tok) * a.hq + head) * D;
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
      // what the scores still want when the maximum is taken; one that underflows (of a q of
      // zeros over 4-bit pages, say) must not make NaN of a masked score's -inf
      const float mul = cap || bias ? 1.f : fmaxf(in_scale, FLT_MIN);
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < x.nblocks; ++j) {
        const int g = g0 + j, sb = g & 1;
        if (!warp_wait(&s_full[sb], (g >> 1) & 1, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        float s[BN];
#pragma unroll
        for (int c = 0; c < BN / 32; ++c)
          tmem_ld_32x32b_x32(lane_base + static_cast<uint32_t>(sb * BN + c * 32), *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
        tmem_ld_wait();

        const int key0 = x.key_of(j);
        if (cap) {
          // a warp whose scores are all far below the cap needs no exponentials for it (16
          // prompts of up to 2048 tokens, cap 30: 450 us, 622 without this branch)
          float far = 0.f;
#pragma unroll
          for (int i = 0; i < BN; ++i) far = fmaxf(far, fabsf(s[i]));
          if (__any_sync(0xffffffffu, !(far * in_scale < 1.f))) {
#pragma unroll
            for (int i = 0; i < BN; ++i) s[i] = capped_score(s[i] * in_scale, cap2);
          } else {
#pragma unroll
            for (int i = 0; i < BN; i += 2) {
              const float2 y = capped_small(make_float2(s[i] * in_scale, s[i + 1] * in_scale), cap2);
              s[i] = y.x;
              s[i + 1] = y.y;
            }
          }
        }
        if (bias) {
          const float first = cap ? 1.f : in_scale, far0 = slope * static_cast<float>(key0 - pos);
#pragma unroll
          for (int i = 0; i < BN; i += 2) {
            const float2 far = fma2(make_float2(slope, slope), make_float2(i, i + 1), make_float2(far0, far0));
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
          if (!warp_wait(o_done, (g - 1) & 1, abort_flag)) {
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
        // V rows that no row of the tile sees may hold anything: a zero weight must meet
        // a zero (converters write zeros there)
        const int z_end = x.kv_len - key0, z_begin = x.key_lo - key0;
        const bool stale = !kFp4 && (z_end < BN || z_begin > 0);
        if (stale) {
          if (!warp_wait(&v_full[g % VST], (g / VST) & 1, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* vt = smem + L::kVOff + (g % VST) * L::kKVBytes;
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
        // one barrier per S buffer: a warp may be a block ahead of another, and its arrival
        // must not stand in for the other's
        if (lane == 0) mbar_arrive(&p_full[sb]);
      }
      // the tile's last P V (o_done may be two phases behind here, o_full completes once a tile)
      if (!ok || !warp_wait(o_full, tile_n & 1, abort_flag)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const bool whole = x.slot < 0;
      const float inv = l > 0.f ? a.v_scale / l : 0.f;
      T* dst = static_cast<T*>(a.out) + (static_cast<int64_t>(x.row0 + x.t0 + tok) * a.hq + head) * D;
      // the part's O, unnormalised, its maximum and sum
      const int64_t part = whole ? 0 : static_cast<int64_t>(x.slot);
      float* part_dst = p.part_o + (part * (D / 4) * BM + row) * 4;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(lane_base + L::kOCol + c, r);
        tmem_ld_wait();
        if (c + 32 == D) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(o_empty);  // the next tile may write O
        }
        if (row >= rows) continue;
        if (whole) {
          uint32_t v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = pack16<T>(__uint_as_float(r[2 * i]) * inv, __uint_as_float(r[2 * i + 1]) * inv);
          if (p.wide_out) {
#pragma unroll
            for (int i = 0; i < 16; i += 8)
              asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst + c + 2 * i), "r"(v[i]), "r"(v[i + 1]),
                           "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
                           : "memory");
          } else {
#pragma unroll
            for (int i = 0; i < 16; i += 4) *reinterpret_cast<uint4*>(dst + c + 2 * i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint4*>(part_dst + (c + i) * BM) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
        }
      }
      if (!whole && row < rows) p.part_ml[part * BM + row] = make_float2(m_used, l);
      g0 += x.nblocks;
      ++tile_n;
    }
    if (!ok && lane == 0) {
      set_device_error(a.seqs.err, kDevErrAttentionTimeout);
      *abort_flag = 1;
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

// Merges the parts of the tiles that were cut, in order. grid = (tiles x D / 16, KV heads,
// sequences); a warp's lanes are rows, a thread takes 4 elements of two chunks. Which
// parts there are is worked out while the main kernel still runs: positions and starts
// were final before that began.
template <typename T, int D>
__global__ void __launch_bounds__(256) attn_paged_prefill_combine_kernel(const PrefillArgs p) {
  constexpr int CHUNKS = D / 16;  // of 16 dims
  const PagedAttnArgs& a = p.a;
  const int chunk = blockIdx.x % CHUNKS, tile = blockIdx.x / CHUNKS, kvh = blockIdx.y, b = blockIdx.z;
  Tile x;
  const int parts = tile_set(p, seq_rows(a.seqs, b, false), b, kvh, tile, x) ? parts_of(p, x.nblocks) : 1;
  const int64_t slot0 = (static_cast<int64_t>(b * a.hkv + kvh) * p.tiles + tile) * p.split;
  pdl_wait();
  pdl_trigger();
  if (parts == 1) return;
  const int r = threadIdx.x & (BM - 1);
  if (r >= x.tokens * a.group) return;
  const int tok = r / a.group, head = kvh * a.group + r - tok * a.group;
  T* dst = static_cast<T*>(a.out) + (static_cast<int64_t>(x.row0 + x.t0 + tok) * a.hq + head) * D;
#pragma unroll
  for (int d4 = chunk * 4 + threadIdx.x / BM; d4 < chunk * 4 + 4; d4 += 2) {
    float top = -INFINITY, den = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < parts; s0 += 4) {
      float2 ml[4];
      float4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        ml[k] = make_float2(-INFINITY, 0.f);
        v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        const int i = s0 + k;
        if (i >= parts) continue;
        const int64_t slot = slot0 + i;
        ml[k] = p.part_ml[slot * BM + r];
        v[k] = *reinterpret_cast<const float4*>(p.part_o + ((slot * (D / 4) + d4) * BM + r) * 4);
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
    const float inv = a.v_scale / den;
    *reinterpret_cast<uint2*>(dst + d4 * 4) = make_uint2(pack16<T>(sum.x * inv, sum.y * inv), pack16<T>(sum.z * inv, sum.w * inv));
  }
}

// ---- host ------------------------------------------------------------------------
struct PrefillPlan {
  int64_t tiles, pairs, units;
  int tile_tokens, pairs_group, split, min_part;
  size_t part_o, workspace;
};

PrefillPlan plan_prefill(int64_t batch, int64_t hkv, int64_t group, int64_t max_new, int64_t head_dim, int64_t max_keys) {
  PrefillPlan p{};
  p.tile_tokens = static_cast<int>(BM / group);
  p.tiles = ceil_div(max_new, p.tile_tokens);
  p.pairs = hkv * batch;
  p.units = p.tiles * p.pairs;
  // pairs of a group: their K and V (2 x 2 bytes an element) within about a quarter of L2
  p.pairs_group = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(p.pairs, (32ll << 20) / (4 * head_dim * std::max<int64_t>(1, max_keys)))));
  // Places for CTAs left over: parts until all have one, of at least 4 key blocks (256
  // keys). With up to two tiles for each place, parts of 1792 keys or more, so that the
  // tiles of the longest sequences do not run on alone: us whole -> in parts, 28/4 heads,
  // 16 x 60 tokens over 16,000 keys 322 -> 206, over 4,000 88 -> 79, 2 x 500 over 10,000
  // 211 -> 127, 64/8 heads 4 x 200 over 20,000 407 -> 371. Smaller parts or more tiles
  // cost more than they level: 4 x 301 over 3,001 65 -> 76, 64 x 60 over 4,000 205 -> 223.
  const int64_t places = 2ll * sm_count();
  p.split = 1;
  p.min_part = 4;
  if (2 * p.units <= places) {
    p.split = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({places / std::max<int64_t>(1, p.units), max_keys / (4 * BN), 64})));
  } else if (p.units <= 2 * places) {
    p.min_part = 28;
    p.split = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(4, max_keys / (28 * BN))));
  }
  if (p.split > 1) {
    p.part_o = static_cast<size_t>(p.units * p.split * BM * head_dim) * 4;
    p.workspace = p.part_o + static_cast<size_t>(p.units * p.split * BM) * 8;
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
  p.tiles = static_cast<int>(plan.tiles);
  p.split = plan.split;
  p.min_part = plan.min_part;
  p.pairs_group = plan.pairs_group;
  p.wide_out = aligned(a.out, 32);
  p.q_bytes = static_cast<unsigned>(plan.tile_tokens * a.group * D * 2);
  if (plan.split > 1) {
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
  launch_pdl(kern, dim3(static_cast<unsigned>(plan.units * plan.split)), dim3(Roles<kFp4>::kThreads), L::kBytes,
             stream, p, tq, tk, tv);
  if (plan.split > 1)
    launch_pdl(attn_paged_prefill_combine_kernel<T, D>,
               dim3(static_cast<unsigned>(plan.tiles * (D / 16)), static_cast<unsigned>(a.hkv),
                    static_cast<unsigned>(a.seqs.batch)),
               dim3(256), 0, stream, p);
  return check_launch("attention_paged", plan.split > 1 ? 2 : 1);
}

int64_t keys_of(const PagedAttnArgs& a) {
  return std::min<int64_t>(a.seqs.max_pages << a.seqs.page_shift, static_cast<int64_t>(a.window) + a.seqs.max_new);
}

}  // namespace

bool paged_prefill_serves(const PagedAttnArgs& a, dli_dtype dtype, dli_dtype kv_dtype) {
  // the grid's x dimension, and int arithmetic on it
  if (a.group > BM || ceil_div(a.seqs.max_new, BM / a.group) * a.hkv * static_cast<int64_t>(a.seqs.batch) > (1ll << 30)) return false;
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
