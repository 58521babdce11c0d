// Decode attention over a prefix that groups of sequences share in the paged cache: every group's prefix is read once for all of its sequences.
//
// With n sequences of a group and G query heads per key head, a prefix of P tokens meets n·G query rows per key head: 2·n·G products per element of K and V
// instead of 2·G per sequence, read n times.  Up to a few hundred rows the keys and values (4·D bytes per token and key head, once per group) are what
// bounds it, so the work is laid out to stream them: an item is up to 128 query rows of one group and a run of 128-token blocks of its prefix, a CTA takes an
// item for one key head, and the items are cut so that they fill the SMs evenly (`ops.shared_prefix`).  Each writes its rows' running maximum, sum and unscaled
// output in fp32.  A second kernel for the sequences' own pages runs beside this one on the same SMs and does likewise; a third joins what both found.
//
// In a CTA the blocks of its run alternate between two streams of their own scores and output in tensor memory, so that the products of one run under
// the softmax of the other; both meet the same query rows and are joined at the end.  Pages are loaded as boxes of up to 128 whole rows of a page (any page size that is a multiple
// of 8): in shared memory eight rows' first 128 bytes lie together, then the same rows' second 128 bytes, then the next eight rows.
// Tensor memory: scores [0,128) and [128,256), both parts of P in place of their scores (32 at a time), output [256,384) and [384,512).
//
// Precision: probabilities go into the product as two bf16 parts, the leading one cut off (not rounded), so that neither part is negative and an infinite
// value comes out as infinity; their sum is within 2^-16 of the value.  The second product costs nothing while memory is the bound.
//
// Measured, 32/8 heads of 128 unless said otherwise, us on the device for all three kernels against reading every page per sequence: 64 sequences of 8 prompts of 0.7–2 k tokens
// with up to 1 k of their own 49 against 77, 128 behind one prompt of 8 k 57 against 504, 13 of one of 32 k (32/4 heads) 31 against 154.  This kernel alone: 43 MB of 8 prompts 20 us, 67 MB of the
// 32 k prompt 22 us (3.0 TB/s).  Of these 2.5 us pass until the first block is there (plan, table and page one after the other from memory), 3 from the last product to the stored results; a block of
// 128 tokens takes 2500 cycles of a CTA, a round of scores, softmax and product in two streams.  That, not memory, bounds 512 rows on one prompt (33 us, 49 % of the tensor pipe).
// Boxes of 16 rows and 128 bytes issued by a lane each took 80 cycles a box, 2600 a block; keys and values behind one producer waited for each other's places; a block's code with all scores in
// registers (10 KB) took 7500 cycles the first time.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/types.h>

#include "common.cuh"
#include "elect.cuh"
#include "host.h"
#include "mma16.cuh"

namespace tk {

using bf16 = __nv_bfloat16;

namespace sp {
constexpr int ROWS = 128, BKV = 128, THREADS = 352, ITEM = 8, JOIN_WARPS = 4;
constexpr int ATOM_BYTES = 128 * 64 * 2;
constexpr float RESCALE_THRESHOLD = 8.f;      // log2 units
template <int D>
struct Smem {
  static constexpr int TILE = D / 64 * ATOM_BYTES, STAGES = D == 128 ? 2 : 4;
  static constexpr int Q = 0, K = TILE, V = K + STAGES * TILE, BAR = V + STAGES * TILE, TOTAL = BAR + 256 + 1024;
  static_assert(ROWS * D * 4 <= STAGES * TILE, "the exchange goes where the keys were");
  static_assert(TOTAL <= 232448, "shared memory of a CTA");
};
}  // namespace sp

// mbar_wait of common.cuh, but a page outside the pool is no reason to give up: its tokens count as zeros.
__device__ __forceinline__ bool shared_wait(uint64_t* bar, uint32_t parity, int* err) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  for (uint32_t it = 0;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 0x3ff) == 0x3ff) {
      if (global_timer_ns() - t0 > 2000000000ull) {
        atomicCAS(err, 0, ERR_ATTN_WAIT);
        return false;
      }
      const int e = *reinterpret_cast<volatile int*>(err);
      if (e != 0 && e != ERR_BOUNDS) return false;       // someone else already gave up
    }
  }
}

struct SharedPrefix {
  const int* items;        // [items][8]: first sequence, sequences, first block of 128 tokens, blocks, tokens of the prefix, slot, first sequence of the group (whose row names the pages)
  const int* tables;
  float* part;             // [slots, hkv, 128, D], four columns c of row r at c ^ (r & 7)
  float2* stat;            // [slots, hkv, 128] maximum (log2 units), sum
  int max_blocks, block_size, box, num_blocks, hkv, G, sequences, slots;
  float scale_log2;
  int* err;
};

template <int D>
__global__ void __launch_bounds__(sp::THREADS, 1)
shared_prefix_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const SharedPrefix p) {
  using namespace sp;
  using S = Smem<D>;
  constexpr int NS = S::STAGES, CH = D / 64;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int* item = p.items + blockIdx.x * ITEM;
  const int row0 = item[0], seqs = item[1], tile0 = item[2], n = item[3], tokens = item[4], slot = item[5], named = item[6], kvh = blockIdx.y;
  if (n <= 0) return;                      // an item that fills up a plan (these come first: as the last of the grid they would keep the next kernel from starting beside the live ones)
  // not a plan for these sequences: rows beyond a slot, sequences, blocks or tokens that are not there (differences only: no sum of a plan's numbers wraps)
  if (seqs < 1 || seqs > ROWS / p.G || row0 < 0 || row0 > p.sequences - seqs || slot < 0 || slot >= p.slots || tokens < 1 || tokens > p.max_blocks * p.block_size || tile0 < 0 ||
      n > (tokens - 1) / BKV + 1 - tile0 || named < 0 || named > row0) {
    if (threadIdx.x == 0) atomicCAS(p.err, 0, ERR_BOUNDS);
    return;
  }

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BAR);
  uint64_t* q_full = bars;                 // 1
  uint64_t* s_full = bars + 1;             // 2 streams each
  uint64_t* p_ready = bars + 3;
  uint64_t* o_done = bars + 5;
  uint64_t* k_full = bars + 7;             // NS stages each
  uint64_t* k_empty = k_full + NS;
  uint64_t* v_full = k_empty + NS;
  uint64_t* v_empty = v_full + NS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_empty + NS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 128);
      mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

  if (warp == 8 || warp == 10) {
    // ------------------------------------------- producers: warp 8 the query and the keys, warp 10 the values
    // A block is up to 16 boxes of 8 rows or more of a page.  Lanes look up a box each, 32 ahead of those that are loaded (the table comes from memory as the pages do); the warp
    // walks the boxes together and one thread issues.  A box past the prefix or outside the pool starts behind the tensor and arrives as zeros.
    const bool keys = warp == 8;
    const CUtensorMap* map = keys ? &tmK : &tmV;
    uint64_t *full = keys ? k_full : v_full, *empty = keys ? k_empty : v_empty;
    uint8_t* tile = smem + (keys ? S::K : S::V);
    const int boxes = BKV / p.box, octets = p.box / 8, outside = p.num_blocks * (p.block_size / 8);
    auto lookup = [&](int box) -> int {
      const int t = tile0 * BKV + box * p.box;
      if (box >= n * boxes || t >= tokens) return outside;
      const int block = p.tables[static_cast<size_t>(named) * p.max_blocks + t / p.block_size];
      if (block < 0 || block >= p.num_blocks) {      // whoever reads the word next raises
        atomicCAS(p.err, 0, ERR_BOUNDS);
        return outside;
      }
      return (block * p.block_size + t % p.block_size) / 8;
    };
    int places = lookup(lane), ahead = lookup(32 + lane), j = 0;
    if (elect_one()) {
      tma_prefetch_desc(map);
      if (keys) {
        mbar_expect_tx(q_full, CH * (ROWS / p.G) * p.G * 128);
#pragma unroll
        for (int i = 0; i < CH; ++i) tma_load_3d(smem + S::Q + i * ATOM_BYTES, &tmQ, q_full, i * 64, kvh * p.G, row0);
      }
    }
    __syncwarp();
    for (; j < n; ++j) {
      const int st = j % NS, from = j * boxes & 31;      // boxes are a power of two: a block's are together
      if (j > 0 && from == 0) {
        places = ahead;
        ahead = lookup(j * boxes + 32 + lane);
      }
      if (j >= NS && !__all_sync(0xffffffffu, shared_wait(&empty[st], (j / NS - 1) & 1, p.err))) break;
      if (elect_one()) mbar_expect_tx(&full[st], S::TILE);
      __syncwarp();
      for (int u = 0; u < boxes; ++u) {
        const int octet = __shfl_sync(0xffffffffu, places, from + u);
        if (elect_one()) tma_load_5d(tile + st * S::TILE + u * octets * CH * 1024, map, &full[st], 0, 0, 0, kvh, octet);
        __syncwarp();
      }
    }
    if (j < n) {       // gave up: nobody may leave while copies are on their way into this CTA's memory
      if (keys) mbar_wait(q_full, 0, nullptr, 0);
      for (int i = max(0, j - NS); i < j; ++i) mbar_wait(&full[i % NS], (i / NS) & 1, nullptr, 0);
    }
  } else if (warp == 9) {
    // ----------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc_s = umma_idesc_bf16(ROWS, BKV, false, false);
    constexpr uint32_t idesc_o = umma_idesc_bf16(ROWS, D, false, true);
    const uint64_t dq = umma_desc(smem_u32(smem + S::Q), 16, 1024);
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, shared_wait(bar, parity, p.err)); };
    auto scores = [&](int j) -> bool {
      const int st = j % NS, t = j & 1;
      if (!wait(&k_full[st], (j / NS) & 1)) return false;
      tc_fence_after();
      const uint64_t dk = umma_desc(smem_u32(smem + S::K + st * S::TILE), 16, CH * 1024);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < CH * 4; ++k)
          umma_bf16(tmem_base + t * 128, dq + (((k >> 2) * ATOM_BYTES + (k & 3) * 32) >> 4), dk + (((k >> 2) * 1024 + (k & 3) * 32) >> 4), idesc_s, k ? 1u : 0u);
        umma_commit(&s_full[t]);
        umma_commit(&k_empty[st]);
      }
      __syncwarp();
      return true;
    };
    bool ok = wait(q_full, 0) && scores(0) && (n < 2 || scores(1));
    for (int j = 0; ok && j < n; ++j) {
      const int st = j % NS, t = j & 1;
      ok = wait(&v_full[st], (j / NS) & 1) && wait(&p_ready[t], (j >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      const uint64_t dv = umma_desc(smem_u32(smem + S::V + st * S::TILE), 1024, CH * 1024);
      if (elect_one()) {
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int k = 0; k < BKV / 16; ++k)
            umma_bf16_ts(tmem_base + 256 + t * 128, tmem_base + t * 128 + (k >> 1) * 32 + part * 16 + (k & 1) * 8, dv + k * (2 * CH * 1024 >> 4), idesc_o, part + k > 0 ? 1u : static_cast<uint32_t>(j > 1));
        umma_commit(&v_empty[st]);
        if (j + 2 >= n) umma_commit(&o_done[t]);
      }
      __syncwarp();
      if (j + 2 < n) ok = scores(j + 2);       // runs after the product that reads P from the same columns
    }
  } else {
    // -------------------------------------------------------------- softmax
    // Warps whose rows no sequence has only keep the products going: what their rows of the output hold is not stored.
    const int t = warp >> 2, row = (warp & 3) * 32 + lane, live = seqs * p.G;
    const bool idle = (warp & 3) * 32 >= live;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem_base + t * 128 + lane_off, to = tmem_base + 256 + t * 128 + lane_off;
    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
    float m = -INFINITY;
    float2 l2 = make_float2(0.f, 0.f);
    bool dead = false;
    for (int j = t; j < n; j += 2) {
      if (!__all_sync(0xffffffffu, shared_wait(&s_full[t], (j >> 1) & 1, p.err))) { dead = true; break; }      // a warp stays together
      if (idle) {
        mbar_arrive(&p_ready[t]);
        continue;
      }
      tc_fence_after();
      // Scores are read twice and a few columns at a time: the code of a block that keeps them in registers is 10 KB, and its first run then waits for every line of it.
      const int left = tokens - (tile0 + j) * BKV;
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
      for (int c = 0; c < 4; c += 2) {
        uint32_t r[2][32];
        tmem_ld32(ts + c * 32, r[0]);
        tmem_ld32(ts + c * 32 + 32, r[1]);
        tmem_ld_wait();
        if (left < BKV) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (c * 32 + i >= left) r[i >> 5][i & 31] = 0xff800000u;      // −∞
        }
#pragma unroll
        for (int i = 0; i < 64; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], __uint_as_float(r[i >> 5][i & 31]));
      }
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2;      // the scale is positive
      float alpha = 1.f;
      bool rescale = false;
      if (mx > m + RESCALE_THRESHOLD || (m == -INFINITY && mx != -INFINITY)) {
        alpha = m == -INFINITY ? 0.f : fast_exp2(m - mx);
        rescale = j > 1;
        m = mx;
        l2.x *= alpha;
        l2.y *= alpha;
      }
      const float sub = m == -INFINITY ? 0.f : m;
      if (__any_sync(0xffffffffu, rescale)) {      // the product before has retired: it was issued ahead of these scores
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          tmem_ld32(to + c * 32, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
          tmem_st32(to + c * 32, r);
        }
        tmem_st_wait();
      }
      const float2 neg = make_float2(-sub, -sub), tiny = make_float2(1.17549435e-38f, 1.17549435e-38f);
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {         // 32 scores become 16 columns of leading parts and 16 of what is left
        uint32_t r[32];
        tmem_ld32(ts + c * 32, r);
        tmem_ld_wait();
        if (left < BKV) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (c * 32 + i >= left) r[i] = 0xff800000u;
        }
        uint32_t parts[32];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 x = fma2(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), scale2, neg);
          const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
          l2 = add2(l2, e);
          const uint32_t a = __float_as_uint(e.x), b = __float_as_uint(e.y);
          parts[i] = __byte_perm(a, b, 0x7632);
          // what was cut off, and never nothing: an infinite value then adds to an infinite sum
          const float2 cut = add2(add2(e, make_float2(__uint_as_float((a & 0xffff0000u) ^ 0x80000000u), __uint_as_float((b & 0xffff0000u) ^ 0x80000000u))), tiny);
          parts[16 + i] = pack_bf16(cut.x, cut.y);
        }
        tmem_st32(ts + c * 32, parts);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_ready[t]);
    }
    // ------------------------------------------------------------- epilogue
    // Each stream hands the other half of its columns over in shared memory, which no copy or product uses any more, and sums the half that it gets, in place; the
    // rows then leave in one copy.  Four columns of row r lie at place c ^ (r & 7), there and in the result: threads with a row each meet all banks.
    float* xo = reinterpret_cast<float*>(smem + S::K);
    float* xs = reinterpret_cast<float*>(smem + S::Q);
    const bool two = n > 1;
    dead = dead || !__all_sync(0xffffffffu, shared_wait(&o_done[0], 0, p.err)) || (two && !__all_sync(0xffffffffu, shared_wait(&o_done[1], 0, p.err)));
    tc_fence_after();
    const float l = l2.x + l2.y;
    auto place = [&](int c) { return reinterpret_cast<float4*>(xo + row * D + ((c ^ (row & 7)) << 2)); };
    xs[t * 2 * ROWS + row] = m;
    xs[(t * 2 + 1) * ROWS + row] = l;
    if (two && !dead) {
#pragma unroll 1
      for (int c = 0; c < D / 64; ++c) {
        const int col = (t ^ 1) * (D / 2) + c * 32;
        uint32_t r[32];
        tmem_ld32(to + col, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *place((col + i) >> 2) = make_float4(__uint_as_float(r[i]), __uint_as_float(r[i + 1]), __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
      }
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    const size_t at = (static_cast<size_t>(slot) * p.hkv + kvh) * ROWS;
    if (!dead) {
      const float m0 = xs[row], l0 = xs[ROWS + row], m1 = two ? xs[2 * ROWS + row] : -INFINITY, l1 = two ? xs[3 * ROWS + row] : 0.f, mm = fmaxf(m0, m1);
      const float a0 = m0 == -INFINITY ? 0.f : fast_exp2(m0 - mm), a1 = m1 == -INFINITY ? 0.f : fast_exp2(m1 - mm);
      const float mine = t == 0 ? a0 : a1, theirs = t == 0 ? a1 : a0;
      if (t == 0 && row < live) p.stat[at + row] = make_float2(mm, l0 * a0 + l1 * a1);
#pragma unroll 1
      for (int c = 0; c < D / 64; ++c) {
        const int col = t * (D / 2) + c * 32;
        // without a second stream its half of the columns comes from the first
        uint32_t r[32];
        tmem_ld32((two ? to : tmem_base + 256 + lane_off) + col, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float s = two ? mine : a0;
          float4 o = make_float4(__uint_as_float(r[i]) * s, __uint_as_float(r[i + 1]) * s, __uint_as_float(r[i + 2]) * s, __uint_as_float(r[i + 3]) * s);
          float4* x = place((col + i) >> 2);
          if (two) o = make_float4(fmaf(x->x, theirs, o.x), fmaf(x->y, theirs, o.y), fmaf(x->z, theirs, o.z), fmaf(x->w, theirs, o.w));
          *x = o;
        }
      }
    }
    fence_proxy_async();
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (threadIdx.x == 0 && !dead) {
      asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(p.part + at * D), "r"(smem_u32(xo)), "r"(live * D * 4) : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // the rest is over when the kernel is
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// A sequence has a part in its group's prefix when it is as long (`r`: its line of the plan); else it attends to all of its own keys.
__device__ __forceinline__ bool has_prefix(const int4& r, int n, int slots, int group) {
  return n >= r.x && r.x >= 0 && r.z > 0 && r.y >= 0 && r.z <= slots - r.y && r.w >= 0 && r.w <= sp::ROWS - group;
}
// The sequences' own pages: a CTA per run of 16 tiles of 16 tokens or more of a sequence, key head and eight query heads; tiles go round robin over its four warps, each with rings of
// two tiles of keys and two of values filled by cp.async.  Products as in paged_decode.cu: heads are rows 0–7, rows 8–15 take what rounding the probabilities left.  Its CTAs fit an SM
// beside one of the prefix kernel's (shared memory, and 200 registers a thread: 3 warps of the other on a scheduler leave no more), so that both stream from memory at once.
// 64 sequences with up to 1 k tokens of their own (134 MB) take 35 us alone (4.3 TB/s): a CTA spends 3 of its 8 us on the way to its first keys (length, table, page).  Runs of 8, 24, 32
// tiles: 53, 49, 50 us for the whole pass of that batch against 49, as a key head per warp without a merge (50).  Persistent warps that walk such runs without a pause took 63 to 77 (four warps per SM do not hide a tile's own
// latency), the same units on the prefix kernel's streams 75 (four live rows of 128 pay for all).
namespace ow {
constexpr int WARPS = 4, TILE = 16, RUN = 16, RUNS = 8, HEADS = 8;
template <int D> constexpr int half_bytes() { return 2 * TILE * D; }            // a tile's keys or values
template <int D> constexpr int smem_bytes() { return WARPS * 4 * half_bytes<D>(); }
}  // namespace ow
// Tiles of 16 tokens that hold the keys first … n of a sequence, and how many of them make a run when there are `runs` CTAs for it
__device__ __forceinline__ int own_tiles(int first, int n) { return n > (first & ~15) ? (n - (first & ~15) + 15) / 16 : 0; }
__device__ __forceinline__ int run_tiles(int tiles, int runs) { return max(ow::RUN, (tiles + runs - 1) / runs); }

struct OwnPages {
  const bf16 *q, *kc, *vc;
  const int *tables, *seq_lens, *rows;
  float* part;             // [runs, B, hq, D] unscaled outputs; a run without tokens writes nothing
  float2* stat;            // [runs, B, hq] maximum (log2 units), sum
  int B, hq, hkv, G, block_size, max_blocks, num_blocks, slots, runs;
  float scale_log2;
  int* err;
};

template <int D>
__global__ void __launch_bounds__(ow::WARPS * 32, 3) own_pages_kernel(const OwnPages p) {
  using namespace ow;
  constexpr int CH = D / 8, RPI = 32 / CH, ROW = 2 * D;      // 16-byte chunks of a row, rows that one load of a warp covers, bytes of a row
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // one CTA sees the prefix kernel end, so that this kernel ends after it
  auto leave = [] {
    if (blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
  };
  const int groups = (p.G + HEADS - 1) / HEADS, kvh = blockIdx.x / groups, g0 = blockIdx.x % groups * HEADS, h0 = kvh * p.G + g0, GH = min(HEADS, p.G - g0), b = blockIdx.y, run = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, hrow = lane >> 2;
  const int4 line = reinterpret_cast<const int4*>(p.rows)[b];
  const int n = min(p.seq_lens[b], p.max_blocks * p.block_size), first = has_prefix(line, n, p.slots, p.G) ? line.x : 0;
  const int total = own_tiles(first, n), per = run_tiles(total, p.runs), tiles = min(per, total - run * per);
  if (tiles <= 0) return leave();
  const int base = (first & ~(TILE - 1)) + run * per * TILE, mine = (tiles - warp + WARPS - 1) / WARPS;

  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t *kring = smem + warp * 4 * half_bytes<D>(), *vring = kring + 2 * half_bytes<D>();
  const int* table = p.tables + static_cast<size_t>(b) * p.max_blocks;
  // row of the pools that holds token (lane & 15) of this warp's tile i, or −1
  auto lookup = [&](int i) -> int {
    const int t = base + (warp + i * WARPS) * TILE + (lane & 15);
    if (i >= mine || t >= n || t < first) return -1;
    const int block = table[t / p.block_size];
    if (block < 0 || block >= p.num_blocks) {      // whoever reads the word next raises
      atomicCAS(p.err, 0, ERR_BOUNDS);
      return -1;
    }
    return block * p.block_size + t % p.block_size;
  };
  // keys or values of a tile; chunks of a row are exchanged so that ldmatrix meets all banks
  auto fetch = [&](const bf16* pool, uint8_t* to, bool live, int rows) {
    if (live) {
#pragma unroll
      for (int k = 0; k < TILE / RPI; ++k) {
        const int r = k * RPI + lane / CH, c = lane % CH, row = __shfl_sync(0xffffffffu, rows, r);
        cp_async16(smem_u32(to) + r * ROW + ((c ^ (r & 7)) << 4), pool + (static_cast<size_t>(max(row, 0)) * p.hkv + kvh) * D + c * 8, row >= 0);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int rows[2] = {lookup(0), lookup(1)}, ahead = lookup(2);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    fetch(p.kc, kring + i * half_bytes<D>(), i < mine, rows[i]);
    fetch(p.vc, vring + i * half_bytes<D>(), i < mine, rows[i]);
  }
  // the heads' rows of A; rows 8–15 are zero for the scores
  uint32_t qa[D / 16][2];
#pragma unroll
  for (int k = 0; k < D / 16; ++k) {
    qa[k][0] = qa[k][1] = 0u;
    if (hrow < GH) {
      const uint32_t* q = reinterpret_cast<const uint32_t*>(p.q + (static_cast<size_t>(b) * p.hq + h0 + hrow) * D + k * 16 + quad * 2);
      qa[k][0] = q[0];
      qa[k][1] = q[4];
    }
  }
  float m = -INFINITY, l = 0.f, acc[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  for (int i = 0; i < mine; ++i) {
    uint8_t *ks = kring + (i & 1) * half_bytes<D>(), *vs = vring + (i & 1) * half_bytes<D>();
    asm volatile("cp.async.wait_group 3;" ::: "memory");
    __syncwarp();
    float s[2][4] = {};
    {
      const int r = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;      // tokens 0–7 chunks 0, 1; tokens 8–15 chunks 0, 1
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t bk[4];
        ldsm4(bk, reinterpret_cast<const bf16*>(ks + r * ROW + (((2 * k + half) ^ (r & 7)) << 4)));
        const uint32_t a[4] = {qa[k][0], 0u, qa[k][1], 0u};
        mma(s[0], a, bk[0], bk[1]);
        mma(s[1], a, bk[2], bk[3]);
      }
    }
    __syncwarp();
    const int places = ahead;               // of the tile after the next, into the places that this one leaves
    ahead = lookup(i + 3);
    fetch(p.kc, ks, i + 2 < mine, places);
    const int t0 = base + (warp + i * WARPS) * TILE + quad * 2;
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = t0 + j * 8 + e;
        s[j][e] = t < n && t >= first ? s[j][e] * p.scale_log2 : -INFINITY;
        mx = fmaxf(mx, s[j][e]);
      }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float mn = fmaxf(m, mx), sub = mn == -INFINITY ? 0.f : mn;
    if (__any_sync(0xffffffffu, mn != m)) {
      const float corr = fast_exp2(m - sub);       // 2^−∞ = 0 before the first key
      l *= corr;
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] *= corr;
    }
    m = mn;
    uint32_t a[4];                                  // leading parts in rows 0–7, remainders in rows 8–15
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float p0 = fast_exp2(s[j][0] - sub), p1 = fast_exp2(s[j][1] - sub);
      l += p0 + p1;
      split2(p0, p1, a[2 * j], a[2 * j + 1]);
    }
    asm volatile("cp.async.wait_group 3;" ::: "memory");
    __syncwarp();
    const int r = lane & 15, half = lane >> 4;     // tokens 0–15 of chunk 2j, tokens 0–15 of chunk 2j + 1
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      uint32_t bv[4];
      ldsm4t(bv, reinterpret_cast<const bf16*>(vs + r * ROW + (((2 * j + half) ^ (r & 7)) << 4)));
      mma(acc[2 * j], a, bv[0], bv[1]);
      mma(acc[2 * j + 1], a, bv[2], bv[3]);
    }
    __syncwarp();
    fetch(p.vc, vs, i + 2 < mine, places);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  __syncthreads();                                  // the rings are free: they take the merge
  float* part = reinterpret_cast<float*>(smem);                       // [WARPS][HEADS][D]
  float* stat = part + WARPS * HEADS * D;                             // [2][WARPS][HEADS] maximum, sum
#pragma unroll
  for (int j = 0; j < D / 8; ++j)
    *reinterpret_cast<float2*>(&part[(warp * HEADS + hrow) * D + j * 8 + quad * 2]) = make_float2(whole(acc[j][0], acc[j][2]), whole(acc[j][1], acc[j][3]));
  if (quad == 0) {
    stat[warp * HEADS + hrow] = m;
    stat[(WARPS + warp) * HEADS + hrow] = l;
  }
  __syncthreads();
  const size_t at = (static_cast<size_t>(run) * p.B + b) * p.hq + h0;
  for (int i = threadIdx.x; i < GH * D; i += WARPS * 32) {
    const int h = i / D;
    float mm = stat[h];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) mm = fmaxf(mm, stat[w * HEADS + h]);
    float o = 0.f, ll = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float mw = stat[w * HEADS + h], c = mw == -INFINITY ? 0.f : fast_exp2(mw - mm);
      o += part[w * HEADS * D + i] * c;
      ll += stat[(WARPS + w) * HEADS + h] * c;
    }
    p.part[at * D + i] = o;
    if (i % D == 0) p.stat[at + h] = make_float2(mm, ll);
  }
  leave();
}

// Joins what the pieces of a prefix and a sequence's own pages found: W warps per query head, each with its share of both.  Two trips to memory bound it (lengths and plan are read before the
// wait, figures and first outputs together after it): 3 us behind the kernels before it; one after the other they took 7.
struct SharedJoin {
  const int *rows, *seq_lens;
  const float *part, *own_part;
  const float2 *stat, *own_stat;
  bf16* out;
  int total, hq, hkv, G, slots, runs, width;      // width: tokens that a row of the table has room for
};

template <int D, int W>
__global__ void __launch_bounds__(sp::JOIN_WARPS * 32) shared_join_kernel(const SharedJoin p) {
  constexpr int E = D / 32, HEADS = sp::JOIN_WARPS / W;      // elements of a lane, heads of a CTA
  __shared__ float s_acc[W > 1 ? W : 1][D + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % W, at = blockIdx.x * HEADS + warp / W;
  if (at >= p.total) return;                  // of one head per CTA all warps leave or none
  const int b = at / p.hq, h = at - b * p.hq, kvh = h / p.G;
  const int4 r = reinterpret_cast<const int4*>(p.rows)[b];      // older than the kernels before this one
  const int n = min(p.seq_lens[b], p.width), slots = has_prefix(r, n, p.slots, p.G) ? r.z : 0, row = r.w + h - kvh * p.G;
  const int own_total = own_tiles(slots > 0 ? r.x : 0, n), per = run_tiles(own_total, p.runs), owns = (own_total + per - 1) / per;
  const size_t found = (static_cast<size_t>(r.y) * p.hkv + kvh) * sp::ROWS + row, next = static_cast<size_t>(p.hkv) * sp::ROWS;
  const int c = lane * E, mine = (slots - part + W - 1) / W, theirs = (owns - part + W - 1) / W;      // this warp's pieces and runs: part, part + W, …
  const float *pieces = p.part + (found + part * next) * D + ((c >> 2 ^ (row & 7)) << 2 | (c & 3)), *runs = p.own_part + (part * static_cast<size_t>(p.total) + at) * D + c;
  const size_t piece = W * next * D, run = W * static_cast<size_t>(p.total) * D;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // lane k holds the figures of the k-th of its own runs, of 32 pieces at a time; the first outputs are asked for with them
  const float2 own = lane < owns ? p.own_stat[lane * static_cast<size_t>(p.total) + at] : make_float2(-INFINITY, 0.f);
  float2 s = lane < mine ? p.stat[found + (part + lane * W) * next] : make_float2(-INFINITY, 0.f);
  constexpr int FIRST = 4;
  float v[2 * FIRST][E];
  auto get = [](float (&to)[E], const float* from) {
    if constexpr (E == 4) *reinterpret_cast<float4*>(to) = *reinterpret_cast<const float4*>(from);
    else *reinterpret_cast<float2*>(to) = *reinterpret_cast<const float2*>(from);
  };
#pragma unroll
  for (int k = 0; k < FIRST; ++k) {
    if (k < mine) get(v[k], pieces + k * piece);
    if (k < theirs) get(v[FIRST + k], runs + k * run);
  }
  float m = fmaxf(own.x, s.x);
  if constexpr (W > 1) {
    for (int k = lane; k < slots; k += 32) m = fmaxf(m, p.stat[found + k * next].x);      // the other warps' too
  } else {
    for (int k = lane + 32; k < slots; k += 32) m = fmaxf(m, p.stat[found + k * next].x);
  }
  m = warp_max(m);
  float acc[E], l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  auto add = [&](const float (&x)[E], float w) {
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(x[e], w, acc[e]);
  };
  for (int k0 = 0; k0 < mine; k0 += 32) {
    if (k0 > 0) s = k0 + lane < mine ? p.stat[found + (part + (k0 + lane) * W) * next] : make_float2(-INFINITY, 0.f);
    const float w = s.x == -INFINITY ? 0.f : fast_exp2(s.x - m);
    l += s.y * w;
    if (k0 == 0) {
#pragma unroll
      for (int k = 0; k < FIRST; ++k)
        if (k < mine) add(v[k], __shfl_sync(0xffffffffu, w, k));
    }
#pragma unroll 8
    for (int k = k0 == 0 ? FIRST : 0; k < min(32, mine - k0); ++k) {
      float x[E];
      get(x, pieces + (k0 + k) * piece);
      add(x, __shfl_sync(0xffffffffu, w, k));
    }
  }
  const float w = own.x == -INFINITY ? 0.f : fast_exp2(own.x - m);
  if (part == 0) l += own.y * w;
  l = warp_sum(l);
#pragma unroll
  for (int k = 0; k < FIRST; ++k)
    if (k < theirs) add(v[FIRST + k], __shfl_sync(0xffffffffu, w, part + k * W));
  for (int k = FIRST; k < theirs; ++k) {
    float x[E];
    get(x, runs + k * run);
    add(x, __shfl_sync(0xffffffffu, w, part + k * W));
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) s_acc[part][c + e] = acc[e];
    if (lane == 0) s_acc[part][D] = l;
    __syncthreads();
    if (part > 0) return;
    for (int i = 1; i < W; ++i) {
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += s_acc[i][c + e];
      l += s_acc[i][D];
    }
  }
  const float scale = l > 0.f ? 1.f / l : l;         // a sum that is not a number stays one
  uint32_t o[E / 2];
#pragma unroll
  for (int e = 0; e < E; e += 2) o[e / 2] = pack_bf16(l == 0.f ? 0.f : acc[e] * scale, l == 0.f ? 0.f : acc[e + 1] * scale);
  bf16* to = p.out + static_cast<size_t>(at) * D + c;
  if constexpr (E == 4) *reinterpret_cast<uint2*>(to) = make_uint2(o[0], o[1]);
  else *reinterpret_cast<uint32_t*>(to) = o[0];
}

template <int D>
static void launch_prefix(const SharedPrefix& p, int64_t items, const CUtensorMap& tq, const CUtensorMap& tk_, const CUtensorMap& tv, cudaStream_t stream) {
  static OncePerDevice limit;
  limit(current_device(), [] {
    TK_CUDA_CHECK(cudaFuncSetAttribute(shared_prefix_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, sp::Smem<D>::TOTAL));
    // an SM that gives this kernel no more than it asks for has no room for the next one's CTAs until it is idle
    TK_CUDA_CHECK(cudaFuncSetAttribute(shared_prefix_kernel<D>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  });
  shared_prefix_kernel<D><<<dim3(items, p.hkv), sp::THREADS, sp::Smem<D>::TOTAL, stream>>>(tq, tk_, tv, p);
  count_launch();
  TK_CUDA_CHECK(cudaGetLastError());
}

// A launch that begins while the one before it on the stream runs
template <typename F, typename P>
static void launch_beside(F kernel, dim3 ctas, int threads, int smem, const P& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = ctas;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  TK_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p));
  count_launch();
}

template <int D>
static void launch_own(const OwnPages& p, cudaStream_t stream) {
  static OncePerDevice limit;
  limit(current_device(), [] {
    TK_CUDA_CHECK(cudaFuncSetAttribute(own_pages_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, ow::smem_bytes<D>()));
    TK_CUDA_CHECK(cudaFuncSetAttribute(own_pages_kernel<D>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  });
  launch_beside(own_pages_kernel<D>, dim3(p.hkv * ((p.G + ow::HEADS - 1) / ow::HEADS), p.B, p.runs), ow::WARPS * 32, ow::smem_bytes<D>(), p, stream);
}

template <int D, int W>
static void launch_join(const SharedJoin& p, cudaStream_t stream) {
  constexpr int HEADS = sp::JOIN_WARPS / W;
  launch_beside(shared_join_kernel<D, W>, dim3((p.total + HEADS - 1) / HEADS), sp::JOIN_WARPS * 32, 0, p, stream);
}

// How a call is laid out: CTAs of a sequence's own part, by what it has room for (where there is more a CTA's run is longer): 256 tokens each, more where that makes over 14 CTAs per SM; and whether
// four warps join a head.  Heads with many pieces are summed by four: 13 sequences with 37 pieces of 32k tokens 35 -> 31 us; with 5 or fewer one warp does (64 sequences 55 against 57).
static std::tuple<int64_t, bool> split_of(int64_t B, int64_t hq, int64_t hkv, int64_t pieces, int64_t room) {
  const int64_t wide = B * hkv * ((hq / hkv + ow::HEADS - 1) / ow::HEADS);
  int64_t runs = std::max<int64_t>(1, std::min<int64_t>(ow::RUNS, (room + ow::RUN * ow::TILE - 1) / (ow::RUN * ow::TILE)));
  while (runs > 1 && wide * runs > 14 * num_sms()) runs = (runs + 1) / 2;
  return {runs, pieces > 8};
}
// The same for whoever captures calls: captures of equal numbers are interchangeable.
std::tuple<int64_t, bool> paged_shared_split(int64_t sequences, int64_t heads, int64_t kv_heads, int64_t pieces, int64_t room) {
  TORCH_CHECK(sequences > 0 && kv_heads > 0 && heads > 0 && heads % kv_heads == 0, "sequences, heads of a multiple of the key heads");
  return split_of(sequences, heads, kv_heads, pieces, room);
}

// One query token per sequence; pieces: slots of a sequence at most; room: tokens that a sequence has at most beside its prefix (what their split is chosen by); plan int32
// [items · 8 + B · 4]: the items, then for every sequence the tokens of its prefix, its first slot, its slots and its row in them.
torch::Tensor paged_attn_shared(const torch::Tensor& q, const torch::Tensor& kc, const torch::Tensor& vc, const torch::Tensor& tables, const torch::Tensor& seq_lens, const torch::Tensor& plan,
                                int64_t items, int64_t slots, int64_t pieces, int64_t room, double scale) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == torch::kBFloat16 && q.is_contiguous() && q.dim() == 3, "q [B,Hq,D] bf16");
  TORCH_CHECK(kc.is_contiguous() && vc.is_contiguous() && kc.dim() == 4 && kc.sizes() == vc.sizes() && kc.scalar_type() == torch::kBFloat16 && vc.scalar_type() == torch::kBFloat16,
              "caches [blocks,bs,Hkv,D] bf16 of one shape");
  const int64_t B = q.size(0), hq = q.size(1), D = q.size(2), hkv = kc.size(2), bs = kc.size(1), G = hkv > 0 ? hq / hkv : 0;
  TORCH_CHECK(kc.size(3) == D && (D == 64 || D == 128) && hkv > 0 && hq % hkv == 0 && G >= 1 && G <= sp::ROWS && bs % 8 == 0 && bs > 0, "heads of 64 or 128, pages of a multiple of 8 tokens");
  TORCH_CHECK(kc.size(0) * bs < (int64_t(1) << 31) - sp::ROWS && hkv * ((G + ow::HEADS - 1) / ow::HEADS) <= 65535 && B <= 65535, "pools of up to 2^31 rows, 65535 sequences");
  for (const auto* t : {&q, &kc, &vc}) TORCH_CHECK(t->device() == q.device() && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0, "q and caches on one device and on 16-byte boundaries");
  for (const auto* t : {&tables, &seq_lens, &plan}) TORCH_CHECK(t->device() == q.device() && t->scalar_type() == torch::kInt32 && t->is_contiguous(), "int32 tables, lengths and plan on the device of q");
  TORCH_CHECK(tables.dim() == 2 && tables.size(0) == B && seq_lens.numel() == B, "a row of the table and a length per sequence");
  TORCH_CHECK(items > 0 && slots > 0 && room >= 0 && plan.numel() == items * sp::ITEM + B * 4, "plan of other sequences");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(plan.data_ptr()) % 16 == 0 && tables.size(1) * bs < (int64_t(1) << 31), "plan on a 16-byte boundary, contexts below 2^31");
  c10::cuda::CUDAGuard guard(q.device());
  auto out = torch::empty_like(q);
  const auto [runs, many] = split_of(B, hq, hkv, pieces, room);
  // one workspace: outputs of the pieces and of the runs, then their figures
  const int64_t pieces_rows = slots * hkv * sp::ROWS, runs_rows = runs * B * hq;
  auto work = torch::empty({(pieces_rows + runs_rows) * (D + 2)}, q.options().dtype(torch::kFloat32));
  float *part = work.data_ptr<float>(), *own_part = part + pieces_rows * D, *stat = own_part + runs_rows * D, *own_stat = stat + pieces_rows * 2;
  const int64_t box = std::min<int64_t>(bs & -bs, sp::BKV);      // the largest power of two that divides a page
  const CUtensorMap tq = make_tmap_3d(q.data_ptr(), D, hq, B, D, hq * D, 64, G, sp::ROWS / G);
  const uint64_t dims[5] = {64, 8, static_cast<uint64_t>(D / 64), static_cast<uint64_t>(hkv), static_cast<uint64_t>(kc.size(0) * bs / 8)};
  const uint64_t strides[4] = {static_cast<uint64_t>(hkv * D), 64, static_cast<uint64_t>(D), static_cast<uint64_t>(8 * hkv * D)};
  const uint32_t boxes[5] = {64, 8, static_cast<uint32_t>(D / 64), 1, static_cast<uint32_t>(box / 8)};
  const CUtensorMap tk_ = make_tmap_5d(kc.data_ptr(), dims, strides, boxes), tv = make_tmap_5d(vc.data_ptr(), dims, strides, boxes);
  SharedPrefix p{};
  p.items = plan.data_ptr<int>(); p.tables = tables.data_ptr<int>(); p.part = part; p.stat = reinterpret_cast<float2*>(stat);
  p.max_blocks = tables.size(1); p.block_size = bs; p.box = box; p.num_blocks = kc.size(0); p.hkv = hkv; p.G = G; p.sequences = B; p.slots = slots;
  p.scale_log2 = static_cast<float>(scale * 1.4426950408889634); p.err = error_word();
  auto stream = at::cuda::getCurrentCUDAStream();
  if (D == 128) launch_prefix<128>(p, items, tq, tk_, tv, stream); else launch_prefix<64>(p, items, tq, tk_, tv, stream);
  const int* rows = plan.data_ptr<int>() + items * sp::ITEM;
  const OwnPages own{reinterpret_cast<const bf16*>(q.data_ptr()), reinterpret_cast<const bf16*>(kc.data_ptr()), reinterpret_cast<const bf16*>(vc.data_ptr()), tables.data_ptr<int>(),
                     seq_lens.data_ptr<int>(), rows, own_part, reinterpret_cast<float2*>(own_stat), static_cast<int>(B), static_cast<int>(hq),
                     static_cast<int>(hkv), static_cast<int>(G), static_cast<int>(bs), static_cast<int>(tables.size(1)), static_cast<int>(kc.size(0)), static_cast<int>(slots), static_cast<int>(runs),
                     p.scale_log2, p.err};
  if (D == 128) launch_own<128>(own, stream); else launch_own<64>(own, stream);
  const SharedJoin join{rows, own.seq_lens, p.part, own.part, p.stat, own.stat, reinterpret_cast<bf16*>(out.data_ptr()), static_cast<int>(B * hq), static_cast<int>(hq), static_cast<int>(hkv),
                        static_cast<int>(G), static_cast<int>(slots), static_cast<int>(runs), static_cast<int>(tables.size(1) * bs)};
  if (D == 128) many ? launch_join<128, 4>(join, stream) : launch_join<128, 1>(join, stream);
  else many ? launch_join<64, 4>(join, stream) : launch_join<64, 1>(join, stream);
  return out;
}

}  // namespace tk
