// Decode attention over a prefix that groups of sequences share in the paged cache: every group's prefix is read once for all of its sequences.
//
// With n sequences of a group and G query heads per key head, a prefix of P tokens meets n·G query rows per key head: 2·n·G products per element of K and V
// instead of 2·G per sequence, read n times.  Up to a few hundred rows the keys and values (4·D bytes per token and key head, once per group) are what
// bounds it, so the work is laid out to stream them: an item is up to 128 query rows of one group and a run of 128-token blocks of its prefix, a CTA takes an
// item for one key head, and the items are cut so that they fill the SMs evenly (`ops.shared_prefix`).  Each writes its rows' running maximum, sum and unscaled
// output in fp32; the decode kernel that reads every sequence's own pages (paged_decode.cu) joins them with what it found itself.
//
// In a CTA the blocks of its run alternate between two streams of their own scores and output in tensor memory, so that the products of one run under
// the softmax of the other; both meet the same query rows and are joined at the end.  Pages are loaded as boxes of up to 128 rows of a page (any page size that is a multiple of 8).
// Tensor memory: scores [0,128) and [128,256), P in place of its scores, output [256,384) and [384,512).
//
// Precision: probabilities go into the product as two bf16 parts, the leading one cut off (not rounded), so that neither part is negative and an infinite
// value comes out as infinity; their sum is within 2^-16 of the value.  The second product costs nothing while memory is the bound.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/types.h>

#include "common.cuh"
#include "elect.cuh"
#include "host.h"
#include "paged_decode.h"

namespace tk {

using bf16 = __nv_bfloat16;

namespace sp {
constexpr int ROWS = 128, BKV = 128, THREADS = 320, ITEM = 8;
constexpr int ATOM_BYTES = 128 * 64 * 2;
constexpr float RESCALE_THRESHOLD = 8.f;      // log2 units
template <int D>
struct Smem {
  static constexpr int TILE = D / 64 * ATOM_BYTES, STAGES = D == 128 ? 3 : 4;
  static constexpr int Q = 0, K = TILE, V = K + STAGES * TILE, BAR = V + STAGES * TILE, STAT = BAR + 256, TOTAL = STAT + 2 * ROWS * 4 + 1024;
  static constexpr int PITCH = D + 4;         // of the exchanged output, in floats: rows on different banks
  static_assert(ROWS * PITCH * 4 <= STAGES * TILE, "the exchange goes where the keys were");
  static_assert(TOTAL <= 232448, "shared memory of a CTA");
};
}  // namespace sp

struct SharedPrefix {
  const int* items;        // [items][8]: first sequence, sequences, first block of 128 tokens, blocks, tokens of the prefix, slot
  const int* tables;
  float* part;             // [slots, hkv, 128, D]
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
  const int row0 = item[0], seqs = item[1], tile0 = item[2], n = item[3], tokens = item[4], slot = item[5], kvh = blockIdx.y;
  if (n <= 0) return;                      // an item that fills up a captured plan
  if (row0 < 0 || row0 >= p.sequences || tile0 < 0 || slot < 0 || slot >= p.slots || tokens > p.max_blocks * p.block_size) {      // not a plan for these sequences
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

  if (warp == 8) {
    // ------------------------------------------------------------- producer
    // Lane = one box of a block's keys and of its values (at most 16 boxes of rows times two chunks of columns).  A box past the prefix or outside the pool starts behind the
    // tensor and arrives as zeros.
    const int boxes = BKV / p.box, unit = lane % boxes, c = lane / boxes;
    const bool mine = c < CH;
    const int outside = p.num_blocks * p.block_size;
    auto lookup = [&](int j) -> int {
      const int t = (tile0 + j) * BKV + unit * p.box;
      if (!mine || j >= n || t >= tokens) return outside;
      const int block = p.tables[static_cast<size_t>(row0) * p.max_blocks + t / p.block_size];
      if (block < 0 || block >= p.num_blocks) {      // whoever reads the word next raises
        atomicCAS(p.err, 0, ERR_BOUNDS);
        return outside;
      }
      return block * p.block_size + t % p.block_size;
    };
    int row = lookup(0), issued = 0;
    if (lane == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      mbar_expect_tx(q_full, CH * (ROWS / p.G) * p.G * 128);
#pragma unroll
      for (int i = 0; i < CH; ++i) tma_load_3d(smem + S::Q + i * ATOM_BYTES, &tmQ, q_full, i * 64, kvh * p.G, row0);
    }
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const int st = j % NS, next = lookup(j + 1);
      if (j >= NS) ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[st], (j / NS - 1) & 1, p.err, ERR_ATTN_WAIT));
      if (!ok) break;
      if (lane == 0) mbar_expect_tx(&k_full[st], S::TILE);
      __syncwarp();
      if (mine) tma_load_3d(smem + S::K + st * S::TILE + c * ATOM_BYTES + unit * p.box * 128, &tmK, &k_full[st], c * 64, kvh, row);
      if (j >= NS) ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[st], (j / NS - 1) & 1, p.err, ERR_ATTN_WAIT));
      if (!ok) {
        mbar_wait(&k_full[st], (j / NS) & 1, nullptr, 0);
        break;
      }
      if (lane == 0) mbar_expect_tx(&v_full[st], S::TILE);
      __syncwarp();
      if (mine) tma_load_3d(smem + S::V + st * S::TILE + c * ATOM_BYTES + unit * p.box * 128, &tmV, &v_full[st], c * 64, kvh, row);
      row = next;
      issued = j + 1;
    }
    if (!ok) {       // nobody may leave while copies are on their way into this CTA's memory
      mbar_wait(q_full, 0, nullptr, 0);
      for (int j = max(0, issued - NS); j < issued; ++j) {
        mbar_wait(&k_full[j % NS], (j / NS) & 1, nullptr, 0);
        mbar_wait(&v_full[j % NS], (j / NS) & 1, nullptr, 0);
      }
    }
  } else if (warp == 9) {
    // ----------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc_s = umma_idesc_bf16(ROWS, BKV, false, false);
    constexpr uint32_t idesc_o = umma_idesc_bf16(ROWS, D, false, true);
    const uint64_t dq = umma_desc(smem_u32(smem + S::Q), 16, 1024);
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.err, ERR_ATTN_WAIT)); };
    auto scores = [&](int j) -> bool {
      const int st = j % NS, t = j & 1;
      if (!wait(&k_full[st], (j / NS) & 1)) return false;
      tc_fence_after();
      const uint64_t dk = umma_desc(smem_u32(smem + S::K + st * S::TILE), 16, 1024);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < CH * 4; ++k) {
          const uint32_t off = ((k >> 2) * ATOM_BYTES + (k & 3) * 32) >> 4;
          umma_bf16(tmem_base + t * 128, dq + off, dk + off, idesc_s, k ? 1u : 0u);
        }
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
      const uint64_t dv = umma_desc(smem_u32(smem + S::V + st * S::TILE), ATOM_BYTES, 1024);
      if (elect_one()) {
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int k = 0; k < BKV / 16; ++k)
            umma_bf16_ts(tmem_base + 256 + t * 128, tmem_base + t * 128 + part * 64 + k * 8, dv + k * (2048 >> 4), idesc_o, part + k > 0 ? 1u : static_cast<uint32_t>(j > 1));
        umma_commit(&v_empty[st]);
        if (j + 2 >= n) umma_commit(&o_done[t]);
      }
      __syncwarp();
      if (j + 2 < n) ok = scores(j + 2);       // runs after the product that reads P from the same columns
    }
  } else {
    // -------------------------------------------------------------- softmax
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem_base + t * 128 + lane_off, to = tmem_base + 256 + t * 128 + lane_off;
    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
    float m = -INFINITY;
    float2 l2 = make_float2(0.f, 0.f);
    bool dead = false;
    for (int j = t; j < n; j += 2) {
      if (!mbar_wait(&s_full[t], (j >> 1) & 1, p.err, ERR_ATTN_WAIT)) { dead = true; break; }
      tc_fence_after();
      float sc[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(ts + c * 32, *reinterpret_cast<uint32_t(*)[32]>(sc + c * 32));
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 128; i += 2) {
        const float2 x = mul2(make_float2(sc[i], sc[i + 1]), scale2);
        sc[i] = x.x;
        sc[i + 1] = x.y;
      }
      const int left = tokens - (tile0 + j) * BKV;
      if (left < BKV) {
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i >= left) sc[i] = -INFINITY;
      }
      float mx4[4] = {sc[0], sc[1], sc[2], sc[3]};
#pragma unroll
      for (int i = 4; i < 128; i += 4) {
        mx4[0] = fmaxf(mx4[0], sc[i]);
        mx4[1] = fmaxf(mx4[1], sc[i + 1]);
        mx4[2] = fmaxf(mx4[2], sc[i + 2]);
        mx4[3] = fmaxf(mx4[3], sc[i + 3]);
      }
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
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
      const float2 neg = make_float2(-sub, -sub);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t lead[32], rest[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float2 x = add2(make_float2(sc[half * 64 + 2 * i], sc[half * 64 + 2 * i + 1]), neg);
          const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
          l2 = add2(l2, e);
          const uint32_t a = __float_as_uint(e.x), b = __float_as_uint(e.y);
          lead[i] = __byte_perm(a, b, 0x7632);
          // what was cut off, and at least 2^-126: an infinite value then adds to an infinite sum
          rest[i] = pack_bf16(fmaxf(e.x - __uint_as_float(a & 0xffff0000u), 1.17549435e-38f), fmaxf(e.y - __uint_as_float(b & 0xffff0000u), 1.17549435e-38f));
        }
        tmem_st32(ts + half * 32, lead);
        tmem_st32(ts + 64 + half * 32, rest);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_ready[t]);
    }
    // ------------------------------------------------------------- epilogue
    // The second stream hands its rows over in shared memory, which no copy or product uses any more; the first writes the sum of both.
    float* xo = reinterpret_cast<float*>(smem + S::K);
    float* xs = reinterpret_cast<float*>(smem + S::STAT);
    const bool two = n > 1;
    dead = dead || !mbar_wait(&o_done[0], 0, p.err, ERR_ATTN_WAIT) || (two && !mbar_wait(&o_done[1], 0, p.err, ERR_ATTN_WAIT));
    tc_fence_after();
    float l = l2.x + l2.y;
    if (t == 1 && two && !dead) {
      xs[row] = m;
      xs[ROWS + row] = l;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        tmem_ld32(to + c * 32, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *reinterpret_cast<float4*>(xo + row * S::PITCH + c * 32 + i) =
              make_float4(__uint_as_float(r[i]), __uint_as_float(r[i + 1]), __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
      }
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (t == 0 && !dead) {
      const float m1 = two ? xs[row] : -INFINITY, l1 = two ? xs[ROWS + row] : 0.f, mm = fmaxf(m, m1);
      const float a0 = m == -INFINITY ? 0.f : fast_exp2(m - mm), a1 = m1 == -INFINITY ? 0.f : fast_exp2(m1 - mm);
      const bool live = row < seqs * p.G;
      const size_t at = (static_cast<size_t>(slot) * p.hkv + kvh) * ROWS + row;
      if (live) p.stat[at] = make_float2(mm, l * a0 + l1 * a1);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        tmem_ld32(to + c * 32, r);
        tmem_ld_wait();
        if (live) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float4 o = make_float4(__uint_as_float(r[i]) * a0, __uint_as_float(r[i + 1]) * a0, __uint_as_float(r[i + 2]) * a0, __uint_as_float(r[i + 3]) * a0);
            if (two) {
              const float4 x = *reinterpret_cast<const float4*>(xo + row * S::PITCH + c * 32 + i);
              o = make_float4(fmaf(x.x, a1, o.x), fmaf(x.y, a1, o.y), fmaf(x.z, a1, o.z), fmaf(x.w, a1, o.w));
            }
            *reinterpret_cast<float4*>(p.part + at * D + c * 32 + i) = o;
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int D>
static void launch_prefix(const SharedPrefix& p, int64_t items, const CUtensorMap& tq, const CUtensorMap& tk_, const CUtensorMap& tv, cudaStream_t stream) {
  static OncePerDevice limit;
  limit(current_device(), [] { TK_CUDA_CHECK(cudaFuncSetAttribute(shared_prefix_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, sp::Smem<D>::TOTAL)); });
  shared_prefix_kernel<D><<<dim3(items, p.hkv), sp::THREADS, sp::Smem<D>::TOTAL, stream>>>(tq, tk_, tv, p);
  count_launch();
  TK_CUDA_CHECK(cudaGetLastError());
}

// One query token per sequence; plan int32 [items · 8 + B · 4]: the items, then for every sequence the tokens of its prefix, its first slot, its slots and its row in them.
torch::Tensor paged_attn_shared(const torch::Tensor& q, const torch::Tensor& kc, const torch::Tensor& vc, const torch::Tensor& tables, const torch::Tensor& seq_lens, const torch::Tensor& plan,
                                int64_t items, int64_t slots, double scale) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == torch::kBFloat16 && q.is_contiguous() && q.dim() == 3, "q [B,Hq,D] bf16");
  TORCH_CHECK(kc.is_contiguous() && vc.is_contiguous() && kc.dim() == 4 && kc.sizes() == vc.sizes() && kc.scalar_type() == torch::kBFloat16 && vc.scalar_type() == torch::kBFloat16,
              "caches [blocks,bs,Hkv,D] bf16 of one shape");
  const int64_t B = q.size(0), hq = q.size(1), D = q.size(2), hkv = kc.size(2), bs = kc.size(1), G = hkv > 0 ? hq / hkv : 0;
  TORCH_CHECK(kc.size(3) == D && (D == 64 || D == 128) && hkv > 0 && hq % hkv == 0 && G >= 1 && G <= sp::ROWS && bs % 8 == 0 && bs > 0, "heads of 64 or 128, pages of a multiple of 8 tokens");
  TORCH_CHECK(kc.size(0) * bs < (int64_t(1) << 31) - sp::ROWS && hkv <= 65535 && B <= 65535, "pools of up to 2^31 rows");
  for (const auto* t : {&q, &kc, &vc}) TORCH_CHECK(t->device() == q.device() && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0, "q and caches on one device and on 16-byte boundaries");
  for (const auto* t : {&tables, &seq_lens, &plan}) TORCH_CHECK(t->device() == q.device() && t->scalar_type() == torch::kInt32 && t->is_contiguous(), "int32 tables, lengths and plan on the device of q");
  TORCH_CHECK(tables.dim() == 2 && tables.size(0) == B && seq_lens.numel() == B, "a row of the table and a length per sequence");
  TORCH_CHECK(items > 0 && slots > 0 && plan.numel() == items * sp::ITEM + B * 4, "plan of other sequences");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(plan.data_ptr()) % 16 == 0 && tables.size(1) * bs < (int64_t(1) << 31), "plan on a 16-byte boundary, contexts below 2^31");
  c10::cuda::CUDAGuard guard(q.device());
  auto out = torch::empty_like(q);
  const auto f32 = q.options().dtype(torch::kFloat32);
  auto part = torch::empty({slots, hkv, sp::ROWS, D}, f32), stat = torch::empty({slots, hkv, sp::ROWS, 2}, f32);
  const int64_t box = std::min<int64_t>(bs & -bs, sp::BKV);      // the largest power of two that divides a page
  const CUtensorMap tq = make_tmap_3d(q.data_ptr(), D, hq, B, D, hq * D, 64, G, sp::ROWS / G);
  const CUtensorMap tk_ = make_tmap_3d(kc.data_ptr(), D, hkv, kc.size(0) * bs, D, hkv * D, 64, 1, box), tv = make_tmap_3d(vc.data_ptr(), D, hkv, kc.size(0) * bs, D, hkv * D, 64, 1, box);
  SharedPrefix p{};
  p.items = plan.data_ptr<int>(); p.tables = tables.data_ptr<int>(); p.part = part.data_ptr<float>(); p.stat = reinterpret_cast<float2*>(stat.data_ptr<float>());
  p.max_blocks = tables.size(1); p.block_size = bs; p.box = box; p.num_blocks = kc.size(0); p.hkv = hkv; p.G = G; p.sequences = B; p.slots = slots;
  p.scale_log2 = static_cast<float>(scale * 1.4426950408889634); p.err = error_word();
  auto stream = at::cuda::getCurrentCUDAStream();
  if (D == 128) launch_prefix<128>(p, items, tq, tk_, tv, stream); else launch_prefix<64>(p, items, tq, tk_, tv, stream);
  const PagedDecode d{q.data_ptr(), kc.data_ptr(), vc.data_ptr(), tables.data_ptr<int>(), seq_lens.data_ptr<int>(), out.data_ptr(), nullptr, OutGate{}, static_cast<int>(hq), static_cast<int>(hkv),
                      static_cast<int>(G), static_cast<int>(bs), static_cast<int>(tables.size(1)), 0, 0, p.scale_log2};
  const PagedJoin join{plan.data_ptr<int>() + items * sp::ITEM, part.data_ptr<float>(), reinterpret_cast<const float2*>(stat.data_ptr<float>()), static_cast<int>(slots), static_cast<int>(kc.size(0)), p.err};
  paged_decode_join(d, join, B, D, stream);
  return out;
}

}  // namespace tk
