// Attention of a batch that shares a long prefix.
//
//   s_j = scale * q . k_j over the prefix keys of the token's group and the visible keys of its own sequence;
//   out = softmax(s) V, as partials (sum_j exp(s_j - m) v_j / l, m + log l) over ranges of keys, joined by their log-sum-exps.
//
// Three kernels.  (1) shared_prefix_kernel, below, reads every prefix once for all the rows of its group: the query rows of a kv head, (token, head of
// the GQA group) pairs of all sequences of the group, are the M rows of tcgen05 products with tiles of 128 keys.  (2) The split-K decode kernel reads
// the sequences' own keys and leaves its partials (decode_splitk.cu).  It runs beside (1), which is bound by the tensor cores where it takes
// long, on the SMs that (1) leaves it.  Or a prefill kernel has left one partial per row, ahead of (1), which then runs beside that one where the caller says that it may (2
// sequences of 14 tokens with 862 and 812 own keys behind 706 keys, 64 heads: 32.0 -> 23.4 us; 4 of 100 tokens behind 3000: 52.5 -> 51.3).  (3) shared_merge_kernel joins the partials
// of a row in a fixed order.
//
// An item of (1) is a block of one or two tiles of 128 rows of one (group, kv head); it takes a step for every 128 keys of the prefix.  The
// steps of all items are dealt out evenly over the CTAs, one per SM, from the lengths on the device (Plan): a CTA has runs of steps
// (segments), each of one item, and writes a partial for each.  The warps of a CTA:
//   warps 0-3 (4-7)  softmax of tile 0 (1), thread = row = lane of tensor memory; they also write the tile's partial
//   then             one warp that copies K and V tiles (TMA; a page, or what a page allows, per copy), one that issues Q K^T, and one
//                    per tile that issues P V with P read from tensor memory
// Up to 128 rows the prefix streams at the rate of the memory; from two tiles on (256 rows are 256 FLOP a byte) the products and
// exponentials of a step take as long as its bytes.  The scores of two tiles take turns in one buffer, so that the tiles stay half a step
// apart; a single tile has two buffers.
//
// Scores, maxima, sums, outputs and all partials are fp32.  One rounding is to 16 bits: the probabilities, to the type of the inputs, as an operand of P V has to be;
// their sum is taken of the unrounded ones (each is off by half a step of bf16 at most, with errors that are independent of one another, so the output is off by
// less than by its own rounding: 0.0023 of its norm together, 0.0017 for that alone).
//
// Keys behind the end of a chunk are masked, their V rows zeroed in shared memory, so what a cache holds there cannot leak.  Every wait is
// bounded; a wait that runs out records a code in the device's status word, and the CTA drains its copies and products, frees its tensor memory and returns.
#include <algorithm>

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"
#include "ptx.cuh"

namespace xfb {
namespace spx {

constexpr int kBM = 128, kBN = 128;          // rows of a query tile, keys of a step
constexpr uint32_t kHalfBytes = 128 * 128;   // a block of 64 columns of a tile
constexpr float kRescaleThreshold = 8.0f;    // a row is re-based when its maximum grew by more than 2^8: probabilities stay below 2^8

struct Args {
  CUtensorMap tm_k, tm_v;  // {D, token rows, kv heads}
  CUtensorMap tm_q;        // {D, q_per_kv, kv heads, tokens}, where a tile is whole tokens (q_tma)
  const void* q;
  float* part_o;    // [slot][slot_rows][D]
  float* part_lse;  // [slot][slot_rows]
  struct GroupPlan* plan;  // [groups], for the merge
  int32_t* status;
  const int32_t* seqstart_q;  // [groups + 1]
  const int32_t* seqlen_k;    // [groups]
  const int32_t* block_tables;
  int64_t bt_stride, kv_rows;
  int64_t q_sm, q_sg, q_sh;
  int32_t groups, kv_heads, q_per_kv, total_q;
  int32_t max_q;         // most tokens of a group
  int32_t kv_bound;      // most keys of a prefix
  int32_t slots, slot_rows;
  int32_t page_size;
  int32_t k_heads_step, v_heads_step;  // 0: all kv heads read the same rows
  int32_t box_tok;       // tokens of a copy: a power of two from 8 to 128
  int32_t q_tma;
  int32_t beside;        // runs beside the kernel ahead in the stream
  float scale_log2;
  uint32_t wait_budget;
  int32_t debug_flags;
};

// How the steps are dealt out.  `aligned`: segments do not cross items -- item i of a group is cut into ceil(steps / share) segments, and CTA c has
// segment c of all of them.  Else, CTA c has the steps [c * share, (c + 1) * share) of all items in a row.  The first costs a CTA one
// prologue and one partial, the second leaves no SM idle.  Where one group has more items than there are CTAs, these come in `waves` first,
// whole items, so that the CTAs go through the keys of a head side by side (the L2 serves all but the first of them; 7016 rows of each of 8 heads
// over 16384 keys, prefix and own keys: 477 us with all steps in a row, 440 so), and only what is left is dealt out by steps.
struct Plan {
  int share, total;  // total: segments (aligned) or steps behind the waves
  int waves;         // whole items of each CTA
  bool aligned;
};
// What the merge has to know of a group: its first segment (aligned) or step, and its first item.
struct GroupPlan {
  int32_t base, item_base;
  int32_t steps;   // per item, 0: no prefix
  int32_t blocks;  // items of a kv head
  int32_t share, aligned, segs, whole;  // segs: segments of an item (aligned); whole: items that are one segment each, ahead of the dealing
};
// A CTA may have this many steps more than the mean before it is worth to let segments cross items (a prologue and an epilogue
// more, which take about as long).
constexpr int kAlignedSlack = 4;

struct Group {
  int q0, rows, steps, klen, blocks;
};
// (A: Args or MergeArgs)
template <typename A>
__device__ __forceinline__ Group group_at(const A& a, int g, int block_rows) {
  // (clamped, so that what it reads and writes stays inside whatever the arrays hold)
  Group r;
  const int q0 = __ldcg(a.seqstart_q + g), q1 = __ldcg(a.seqstart_q + g + 1), len = __ldcg(a.seqlen_k + g);
  r.q0 = min(max(q0, 0), a.total_q);
  r.rows = min(min(max(q1 - r.q0, 0), a.max_q), a.total_q - r.q0) * a.q_per_kv;
  r.klen = min(max(len, 0), a.kv_bound);
  r.steps = r.rows > 0 ? (r.klen + kBN - 1) / kBN : 0;
  r.blocks = (r.rows + block_rows - 1) / block_rows;
  return r;
}
template <typename A>
__device__ __forceinline__ int items_of(const A& a, const Group& g) { return g.steps > 0 ? g.blocks * a.kv_heads : 0; }
__device__ __forceinline__ Plan plan_of_one(int items, int steps, int ctas) {
  if (items == 0) return {1, 0, 0, true};
  const int waves = items / ctas;
  if (waves > 0) {
    const int left = (items - waves * ctas) * steps;
    return {max(1, (left + ctas - 1) / ctas), left, waves, false};
  }
  const int cut = ctas / items, share = (steps + cut - 1) / cut, mean = (items * steps + ctas - 1) / ctas;
  if (share <= mean + kAlignedSlack) return {share, items * ((steps + share - 1) / share), 0, true};
  return {mean, items * steps, 0, false};
}
// `mine`: the group of this lane among the first 32, nothing in the lanes behind the last.  By a whole warp.
__device__ __forceinline__ Plan make_plan(const Args& a, int block_rows, const Group& mine, int lane) {
  const int ctas = gridDim.x;
  if (a.groups == 1) {
    return plan_of_one(__shfl_sync(0xffffffffu, items_of(a, mine), 0), __shfl_sync(0xffffffffu, mine.steps, 0), ctas);
  }
  constexpr int N = kAlignedSlack + 1;
  int steps = 0, sum[N];
  for (int g0 = 0; g0 < a.groups; g0 += 32) {
    const Group g = g0 == 0 ? mine : g0 + lane < a.groups ? group_at(a, g0 + lane, block_rows) : Group{};
    steps += items_of(a, g) * g.steps;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) steps += __shfl_xor_sync(0xffffffffu, steps, o);
  const int mean = max(1, (steps + ctas - 1) / ctas);
#pragma unroll
  for (int i = 0; i < N; ++i) sum[i] = 0;
  for (int g0 = 0; g0 < a.groups; g0 += 32) {
    const Group g = g0 == 0 ? mine : g0 + lane < a.groups ? group_at(a, g0 + lane, block_rows) : Group{};
    const int items = items_of(a, g);
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] += items * ((g.steps + mean + i - 1) / (mean + i));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
  Plan plan = {mean, steps, 0, false};
#pragma unroll
  for (int i = N - 1; i >= 0; --i)
    if (sum[i] <= ctas) plan = {mean + i, sum[i], 0, true};
  return plan;
}

template <int D, int kTiles>
struct Smem {
  static constexpr int kTile = kBM * D * 2;
  static constexpr int kStages = D == 64 ? 4 : kTiles == 2 ? 2 : 3;  // depth of the K and of the V ring
  static constexpr int kQ = 0;
  static constexpr int kK = kTiles * kTile;
  static constexpr int kV = kK + kStages * kTile;
  static constexpr int kBar = kV + kStages * kTile;
  static constexpr int kTotal = kBar + 1024 + 1024;  // (aligned to 1024 bytes inside)
  static_assert(kTotal <= 227 * 1024, "shared memory of one CTA");
};

// A run of steps of one item, as its CTA's warps see it; no steps: none.
struct Segment {
  int g, head, q0, row0, rows, klen, step0, steps, slot, tiles, next;
};

struct __align__(8) Barriers {
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t q_full, q_empty;
  uint64_t s_full[2], s_empty[2];
  uint64_t p_half[2], p_full[2], pv_done[2];
  uint64_t drain[3];
  Segment segment[2];  // this one and the next one
  uint32_t tmem_base;
  uint32_t abort_flag;
};
static_assert(sizeof(Barriers) <= 1024, "barrier block");

// Columns of the tensor memory: scores (one buffer for two tiles, two for one), probabilities (16-bit pairs), output.
template <int D, int kTiles>
struct Tmem {
  __device__ static constexpr uint32_t s(int buf) { return kTiles == 2 ? 0 : buf * kBN; }
  __device__ static constexpr uint32_t p(int t) { return kTiles == 2 ? kBN + t * (kBN / 2) : 2 * kBN; }
  __device__ static constexpr uint32_t o(int t) { return kTiles == 2 ? 2 * kBN + t * D : 2 * kBN + kBN / 2; }
};

__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  if constexpr (kBf16) {
    __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&t);
  } else {
    __half2 t = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&t);
  }
}

__host__ __device__ constexpr int threads(int tiles) { return tiles == 2 ? 384 : 256; }
// registers per thread of the two-tile form after setmaxnreg; their sum must fit what the CTA was launched with
constexpr int kRegsLaunch = 168, kRegsSoftmax = 200, kRegsAux = 104;
static_assert(8 * kRegsSoftmax + 4 * kRegsAux <= 12 * kRegsLaunch, "setmaxnreg would ask for more registers than the CTA owns");

template <int D, bool kBf16, int kTiles>
__global__ void __launch_bounds__(threads(kTiles), 1) shared_prefix_kernel(const __grid_constant__ Args a) {
  using L = Smem<D, kTiles>;
  using T = Tmem<D, kTiles>;
  constexpr int kHalves = D / 64, kTmaWarp = 4 * kTiles, kQkWarp = kTmaWarp + 1, kPvWarp0 = kTmaWarp + 2;
  extern __shared__ uint8_t smem_dyn[];
  uint8_t* smem = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
  Barriers* bar = reinterpret_cast<Barriers*>(smem + L::kBar);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t budget = a.wait_budget;

  // (barriers, tensor memory and its allocation do not wait for the kernel ahead in the stream; everything below does)
  if (warp == kPvWarp0) {
    tmem_alloc(&bar->tmem_base, 512);
    tmem_relinquish();
  } else if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&bar->k_full[i], 1), mbar_init(&bar->k_empty[i], 1);
      mbar_init(&bar->v_full[i], 1), mbar_init(&bar->v_empty[i], kTiles);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bar->s_full[t], 1), mbar_init(&bar->s_empty[t], 4);
      mbar_init(&bar->p_half[t], 4), mbar_init(&bar->p_full[t], 4), mbar_init(&bar->pv_done[t], 1);
    }
    mbar_init(&bar->q_full, 1), mbar_init(&bar->q_empty, 4 * kTiles);
    for (int i = 0; i < 3; ++i) mbar_init(&bar->drain[i], 1);
    bar->abort_flag = 0;
    mbar_fence_init();
  } else if (warp == kTmaWarp && elect_one()) {
    prefetch_tensormap(&a.tm_k), prefetch_tensormap(&a.tm_v);
    if (a.q_tma) prefetch_tensormap(&a.tm_q);
  }
  __syncwarp();
  // Beside the kernel ahead (xfb200_shared_prefix_params.own_beside): everything this one reads was complete when that one began.  The last CTA waits for it at its
  // end, so that whoever waits for this kernel has both.
  if (a.beside)
    beside_fence();
  else
    grid_dep_wait();
  grid_dep_launch();

  constexpr int kBlockRows = kTiles * kBM;
  const int ctas = gridDim.x, cta = blockIdx.x;
  // The copy warp and the Q K^T warp know the plan; the others get their segments from the latter.
  Plan plan{};
  Group mine{};
  // The segment at position `pos`.  Positions of a CTA: -waves .. -1 whole items, then its place in the row of all segments (aligned) or steps.
  auto segment_at = [&](int pos) -> Segment {
    Segment r{};
    const int pos_first = plan.aligned ? cta : cta * plan.share, pos_end = min(pos_first + (plan.aligned ? 1 : plan.share), plan.total);
    if (pos >= 0 && pos >= pos_end) return r;
    int base = 0, item_base = 0;
    for (int g0 = 0;; g0 += 32) {
      const Group g = g0 == 0 ? mine : g0 + lane < a.groups ? group_at(a, g0 + lane, kBlockRows) : Group{};
      const int items = items_of(a, g), per = plan.aligned ? (g.steps + plan.share - 1) / plan.share : g.steps, len = items * per;
      int incl = len, incl_items = items, at = 0;
      if (a.groups > 1) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, incl, o), y = __shfl_up_sync(0xffffffffu, incl_items, o);
          if (lane >= o) incl += x, incl_items += y;
        }
        const uint32_t beyond = __ballot_sync(0xffffffffu, base + incl > pos);
        if (beyond == 0 && g0 + 32 < a.groups) {
          base += __shfl_sync(0xffffffffu, incl, 31), item_base += __shfl_sync(0xffffffffu, incl_items, 31);
          continue;
        }
        at = __ffs(beyond) - 1;  // (there is one: pos is below the total)
      }
      auto from = [&](int x) { return __shfl_sync(0xffffffffu, x, at); };
      const int per_item = from(per), steps = from(g.steps), blocks = from(g.blocks);
      int item, in_item = 0;
      r.steps = steps;
      if (pos < 0) {
        item = (pos + plan.waves) * ctas + cta;
        r.slot = item;
        r.next = pos < -1 ? pos + 1 : pos_first;
      } else {
        const int rel = pos - from(base + incl - len);
        item = rel / per_item, in_item = rel - item * per_item;
        r.step0 = plan.aligned ? in_item * plan.share : in_item;
        r.steps = min(steps - r.step0, plan.aligned ? plan.share : pos_end - pos);
        item += plan.waves * ctas;
        r.slot = plan.aligned ? pos : from(item_base + incl_items - items) + item + cta;
        r.next = plan.aligned ? plan.total : pos + r.steps;
      }
      r.g = g0 + at, r.q0 = from(g.q0), r.rows = from(g.rows), r.klen = from(g.klen);
      r.head = item / blocks, r.row0 = (item - r.head * blocks) * kBlockRows;
      r.tiles = kTiles == 1 || r.rows - r.row0 <= kBM ? 1 : 2;
      return r;
    }
  };
  Segment sg{};
  if (warp == kTmaWarp || warp == kQkWarp) {
    if (lane < a.groups) mine = group_at(a, lane, kBlockRows);
    plan = make_plan(a, kBlockRows, mine, lane);
    sg = segment_at(plan.waves > 0 ? -plan.waves : plan.aligned ? cta : cta * plan.share);
    if (warp == kQkWarp && lane == 0) bar->segment[0] = sg;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar->tmem_base;
  volatile uint32_t* abort_flag = &bar->abort_flag;
  int code = 0;
  auto give_up = [&]() {
    if (lane == 0) atomicCAS(a.status, 0, code);
    *abort_flag = 1;
  };

  // All warps but the copy warp meet twice a segment: behind the load of Q, and at the segment's end, when the next one's Q may be written (every
  // product with this one's is through) and O overwritten (it is read).  There they agree on whether a wait of any of them ran out.
  constexpr int kOthers = threads(kTiles) - 32;
  auto q_loaded = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(kOthers) : "memory"); };  // (Q stored by the softmax warps)
  auto segment_done = [&]() -> bool {
    if (code != 0) give_up();
    int stop;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.s32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, 2, %2, p;\n\t"
        "selp.s32 %0, 1, 0, q;\n\t}\n"
        : "=r"(stop)
        : "r"(code), "n"(kOthers)
        : "memory");
    tc_fence_after();
    return stop == 0;
  };
  // Shared-memory descriptors of the products: the upper word is constant, the lower one holds address >> 4 and the leading-dimension offset.
  constexpr uint32_t kDescHi = 64u | (1u << 14) | (2u << 29);  // stride between 8-row groups 1024 B, version 1, 128B swizzle
  auto desc = [](uint32_t lo_word) -> uint64_t {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo_word), "r"(kDescHi));
    return d;
  };

  if (warp >= kTmaWarp) {
    if constexpr (kTiles == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsAux));
    if (warp == kTmaWarp) {
      // ================================================================== copies
      // A tile is 128 / box_tok copies per half, a lane each; the row of a lane's copy is looked up a step ahead.  V of a step is loaded behind K of
      // the step after it: its stage comes free a softmax later than the K stage, which must not wait for that.
      const int box = a.box_tok, n_box = kBN / box;
      auto row_of = [&](const Segment& sg, int step) -> int {
        const int t = step * kBN + min(lane, n_box - 1) * box;
        if (t >= sg.klen) return 0;
        int64_t row = int64_t(sg.g) * a.kv_bound + t;
        if (a.block_tables != nullptr) {
          const int pg = t / a.page_size;
          row = int64_t(__ldcg(a.block_tables + int64_t(sg.g) * a.bt_stride + pg)) * a.page_size + (t - pg * a.page_size);
        }
        return int(row < 0 || row > a.kv_rows ? a.kv_rows : row);  // (a page outside the pool reads as zero)
      };
      auto load = [&](int at, const CUtensorMap* tm, uint64_t* full, int live, int row, int head) {
        if (lane == 0) mbar_expect_tx(full, uint32_t(live) * box * D * 2);
        __syncwarp();
        if (lane < live) {
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf) tma_load_3d(smem + at + hf * kHalfBytes + lane * box * 128, tm, full, hf * 64, row, head);
        }
        __syncwarp();
      };
      int nk = 0, nv = 0;  // loads issued
      int segments = 0;    // whose Q is
      bool pending = false;
      int v_row = 0, v_head = 0, v_live = 0;
      auto load_v = [&]() -> bool {
        if (!pending) return true;
        const int st = nv % L::kStages;
        if (!mbar_wait(&bar->v_empty[st], ((nv / L::kStages) & 1) ^ 1, abort_flag, budget)) {
          code = 51;
          return false;
        }
        load(L::kV + st * L::kTile, &a.tm_v, &bar->v_full[st], v_live, v_row, v_head);
        ++nv, pending = false;
        return true;
      };
      for (; sg.steps > 0 && code == 0; sg = segment_at(sg.next)) {
        int row = row_of(sg, sg.step0);
        for (int j = sg.step0; j < sg.step0 + sg.steps; ++j) {
          const int st = nk % L::kStages;
          const int next = row_of(sg, j + 1);
          if (!mbar_wait(&bar->k_empty[st], ((nk / L::kStages) & 1) ^ 1, abort_flag, budget)) {
            code = 50;
            break;
          }
          const int live = min(n_box, (sg.klen - j * kBN + box - 1) / box);
          // (testing aid: the first CTA leaves out its first K tile, so that the wait for it runs out)
          if (!((a.debug_flags & 1) && blockIdx.x == 0)) {
            load(L::kK + st * L::kTile, &a.tm_k, &bar->k_full[st], live, row, sg.head * a.k_heads_step);
            ++nk;
          }
          if (!load_v()) break;
          if (a.q_tma && j == sg.step0) {
            // Q behind the first K and the last V of the segment before: its place comes free when the rows of that one have left through it
            if (!mbar_wait(&bar->q_empty, (segments & 1) ^ 1, abort_flag, budget)) {
              code = 49;
              break;
            }
            if (lane == 0) mbar_expect_tx(&bar->q_full, sg.tiles * L::kTile);
            __syncwarp();
            if (lane < sg.tiles * kHalves)
              tma_load_4d(smem + L::kQ + lane * kHalfBytes, &a.tm_q, &bar->q_full, lane % kHalves * 64, 0, sg.head, sg.q0 + (sg.row0 + lane / kHalves * kBM) / a.q_per_kv);
            __syncwarp();
            ++segments;
          }
          pending = true, v_row = row, v_head = sg.head * a.v_heads_step, v_live = live;
          row = next;
        }
      }
      if (code == 0) load_v();
      // what is still in flight has to land before the CTA leaves
      for (int i = max(0, nk - L::kStages); i < nk; ++i) mbar_wait(&bar->k_full[i % L::kStages], (i / L::kStages) & 1, nullptr, budget);
      if (segments > 0) mbar_wait(&bar->q_full, (segments - 1) & 1, nullptr, budget);
      for (int i = max(0, nv - L::kStages); i < nv; ++i) mbar_wait(&bar->v_full[i % L::kStages], (i / L::kStages) & 1, nullptr, budget);
      if (code != 0) give_up();
    } else {
      int n = 0;    // steps so far, over all segments
      int cnt = 0;  // products so far (PV warps: of their tile)
      int n_seg = 0;
      for (int at = 0;; at ^= 1) {
        if (warp != kQkWarp) sg = bar->segment[at];
        const int tiles = sg.tiles, n_steps = sg.steps;
        if (n_steps <= 0) break;
        if (!a.q_tma) q_loaded();
        if (warp == kQkWarp) {
          // ============================================================ Q K^T
          constexpr uint32_t idesc = umma_idesc(kBM, kBN, kBf16, false, false);
          const uint32_t q_lo = (smem_u32(smem + L::kQ) >> 4) | (1u << 16), k_lo = (smem_u32(smem + L::kK) >> 4) | (1u << 16);
          if (a.q_tma && !mbar_wait(&bar->q_full, n_seg++ & 1, abort_flag, budget)) code = 48;
          for (int j = 0; j < n_steps && code == 0; ++j, ++n) {
            const int st = n % L::kStages;
            if (!mbar_wait(&bar->k_full[st], (n / L::kStages) & 1, abort_flag, budget)) {
              code = 52;
              break;
            }
#pragma unroll 1
            for (int t = 0; t < tiles; ++t, ++cnt) {
              const int buf = kTiles == 2 ? 0 : cnt & 1;
              if (!mbar_wait(&bar->s_empty[buf], ((kTiles == 2 ? cnt : cnt >> 1) & 1) ^ 1, abort_flag, budget)) {
                code = 53;
                break;
              }
              tc_fence_after();
              if (elect_one()) {
                uint32_t ql = q_lo + t * (L::kTile >> 4), kl = k_lo + st * (L::kTile >> 4);
#pragma unroll 1
                for (int hf = 0; hf < kHalves; ++hf) {
#pragma unroll
                  for (int kk = 0; kk < 4; ++kk) umma_ss(tmem + T::s(buf), desc(ql + kk * 2), desc(kl + kk * 2), idesc, kk > 0 ? 1u : uint32_t(hf));
                  ql += kHalfBytes >> 4, kl += kHalfBytes >> 4;
                }
                tc_commit(&bar->s_full[kTiles == 2 ? t : buf]);
              }
              __syncwarp();
            }
            if (elect_one()) tc_commit(&bar->k_empty[st]);
          }
          sg = segment_at(sg.next);
          if (lane == 0) bar->segment[at ^ 1] = sg;
        } else if (warp < kPvWarp0 + kTiles) {
          // ============================================================== P V
          const int t = warp - kPvWarp0;
          constexpr uint32_t idesc = umma_idesc(kBM, D, kBf16, false, true);
          const uint32_t v_lo = (smem_u32(smem + L::kV) >> 4) | ((kHalfBytes >> 4) << 16);
          const uint32_t tp = tmem + T::p(t), to = tmem + T::o(t);
          for (int j = 0; j < n_steps && code == 0; ++j, ++n) {
            const int st = n % L::kStages;
            if (!mbar_wait(&bar->v_full[st], (n / L::kStages) & 1, abort_flag, budget)) {
              code = 54;
              break;
            }
            if (t < tiles) {
              const int left = sg.klen - (sg.step0 + j) * kBN;
              if (left < kBN) {
                // V rows past the end may hold anything; P is 0 there.  (Two PV warps write the same zeros: no order between them is needed.)
                uint8_t* vt = smem + L::kV + st * L::kTile;
#pragma unroll 1
                for (int hf = 0; hf < kHalves; ++hf)
#pragma unroll 1
                  for (int i = left * 8 + lane; i < kBN * 8; i += 32) *reinterpret_cast<uint4*>(vt + hf * kHalfBytes + i * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
                __syncwarp();
              }
              uint32_t vl = v_lo + st * (L::kTile >> 4), pt = tp;
#pragma unroll 1
              for (int half = 0; half < 2; ++half) {
                if (!mbar_wait(half == 0 ? &bar->p_half[t] : &bar->p_full[t], cnt & 1, abort_flag, budget)) {
                  code = 55 + t;
                  break;
                }
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                  for (int kk = 0; kk < kBN / 32; ++kk) umma_ts(to, pt + kk * 8, desc(vl + ((kk * 16 * 128) >> 4)), idesc, kk > 0 ? 1u : uint32_t(j > 0 || half > 0));
                  if (half > 0) tc_commit(&bar->pv_done[t]);
                }
                __syncwarp();
                vl += (64 * 128) >> 4, pt += 32;
              }
              ++cnt;
            }
            if (elect_one()) tc_commit(&bar->v_empty[st]);
          }
        }
        if (!segment_done()) break;
      }
      if (cta == 0 && warp == kQkWarp && a.groups > 1) {  // what the merge has to know
        int base = 0, item_base = 0;
        for (int g0 = 0; g0 < a.groups; g0 += 32) {
          const Group g = g0 == 0 ? mine : g0 + lane < a.groups ? group_at(a, g0 + lane, kBlockRows) : Group{};
          const int items = items_of(a, g), segs = (g.steps + plan.share - 1) / plan.share;
          const int len = items * (plan.aligned ? segs : g.steps);
          int incl = len, incl_items = items;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, incl, o), y = __shfl_up_sync(0xffffffffu, incl_items, o);
            if (lane >= o) incl += x, incl_items += y;
          }
          if (g0 + lane < a.groups) a.plan[g0 + lane] = {base + incl - len, item_base + incl_items - items, g.steps, g.blocks, plan.share, plan.aligned, segs, plan.waves * ctas};
          base += __shfl_sync(0xffffffffu, incl, 31), item_base += __shfl_sync(0xffffffffu, incl_items, 31);
        }
      }
      if (warp < kPvWarp0 + kTiles) {
        // products still in flight (after a wait that ran out) have to end before the tensor memory is freed
        uint64_t* drain = &bar->drain[warp - kQkWarp];
        if (elect_one()) tc_commit(drain);
        __syncwarp();
        mbar_wait(drain, 0, nullptr, budget);
      }
    }
  } else {
    // ================================================================ softmax
    if constexpr (kTiles == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    int cnt = 0;  // products of this tile so far
    for (int at = 0;; at ^= 1) {
      const Segment sg = bar->segment[at];
      const int tiles = sg.tiles, n_steps = sg.steps;
      if (n_steps <= 0) break;
      // Where a tile is no whole number of tokens: Q's rows (token, head) in 16-byte chunks, to where the 128-byte swizzle has them; rows past the end are zero.  A thread keeps its column and
      // asks for all its chunks before it stores the first.  (One after the other they took 10 us of a segment.)
      if (!a.q_tma) {
        constexpr int kCols = D / 8, kStride = kBM / kCols, kPer = kBM / kStride;  // threads to a row; rows between two of a thread's; its rows in a tile
        const int c = threadIdx.x % kCols, r0 = (threadIdx.x % kBM) / kCols, t = warp >> 2;
        const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + int64_t(sg.q0) * a.q_sm + int64_t(sg.head) * a.q_sg + c * 8;
        uint4 x[kPer];
        int row = sg.row0 + t * kBM + r0, tok = row / a.q_per_kv, h = row - tok * a.q_per_kv;
        const int step_tok = kStride / a.q_per_kv, step_h = kStride - step_tok * a.q_per_kv;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          x[i] = make_uint4(0, 0, 0, 0);
          if (row < sg.rows) x[i] = __ldcg(reinterpret_cast<const uint4*>(src + int64_t(tok) * a.q_sm + int64_t(h) * a.q_sh));
          row += kStride, tok += step_tok, h += step_h;
          if (h >= a.q_per_kv) h -= a.q_per_kv, ++tok;
        }
        uint8_t* dst = smem + L::kQ + t * L::kTile + (c >> 3) * kHalfBytes;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int rt = r0 + i * kStride;
          *reinterpret_cast<uint4*>(dst + rt * 128 + (((c & 7) ^ (rt & 7)) << 4)) = x[i];
        }
        fence_proxy_async_smem();
        q_loaded();
      }
      if ((warp >> 2) < tiles) {
        const int t = warp >> 2;
        const uint32_t lane_sel = uint32_t((warp & 3) * 32) << 16;
        const uint32_t tmem_p = tmem + T::p(t) + lane_sel, tmem_o = tmem + T::o(t) + lane_sel;
        const uint64_t sc2 = f2_pack(a.scale_log2, a.scale_log2);
        float m_run = -INFINITY, l_run = 0.f;
        auto chunk_max = [](const float* sc) -> float {
          float m0 = fmax3(sc[0], sc[1], sc[2]), m1 = fmax3(sc[3], sc[4], sc[5]), m2 = fmax3(sc[6], sc[7], sc[8]), m3 = fmax3(sc[9], sc[10], sc[11]);
          m0 = fmax3(m0, sc[12], sc[13]), m1 = fmax3(m1, sc[14], sc[15]), m2 = fmax3(m2, sc[16], sc[17]), m3 = fmax3(m3, sc[18], sc[19]);
          m0 = fmax3(m0, sc[20], sc[21]), m1 = fmax3(m1, sc[22], sc[23]), m2 = fmax3(m2, sc[24], sc[25]), m3 = fmax3(m3, sc[26], sc[27]);
          m0 = fmax3(m0, sc[28], sc[29]), m1 = fmax3(m1, sc[30], sc[31]);
          return fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
        };
        auto exp_store = [&](const uint32_t* sr, int col, uint64_t nm2, uint64_t (&sum2)[4]) {
          uint32_t pr[16];
#pragma unroll
          for (int h = 0; h < 32; h += 16) {
            float e[16];
#pragma unroll
            for (int i = 0; i < 16; i += 2) f2_unpack(ffma2(f2_pack(__uint_as_float(sr[h + i]), __uint_as_float(sr[h + i + 1])), sc2, nm2), e[i], e[i + 1]);
#pragma unroll
            for (int i = 0; i < 16; ++i) e[i] = fast_exp2(e[i]);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              sum2[(i / 2) & 3] = fadd2(sum2[(i / 2) & 3], f2_pack(e[i], e[i + 1]));
              pr[(h + i) / 2] = pack_pair<kBf16>(e[i], e[i + 1]);
            }
          }
          XFB_TMEM_ST_16(tmem_p + col, pr);
        };
        for (int j = 0; j < n_steps; ++j, ++cnt) {
          const int buf = kTiles == 2 ? 0 : cnt & 1;
          const uint32_t tmem_s = tmem + T::s(buf) + lane_sel;
          if (!mbar_wait(&bar->s_full[kTiles == 2 ? t : buf], (kTiles == 2 ? cnt : cnt >> 1) & 1, abort_flag, budget)) {
            code = 57 + t;
            break;
          }
          tc_fence_after();
          const int left = sg.klen - (sg.step0 + j) * kBN;  // keys from here to the end of the prefix
          if (left < kBN) {
            // hidden scores become -inf where they lie, so that the step is one piece of code
            uint32_t sm[32];
#pragma unroll 1
            for (int c = left / 32; c < kBN / 32; ++c) {
              const int vis = left - c * 32;
              XFB_TMEM_LD_32(tmem_s + c * 32, sm);
              XFB_TMEM_WAIT_LD_32(sm);
#pragma unroll
              for (int i = 0; i < 32; ++i) sm[i] = i < vis ? sm[i] : 0xff800000u;
              XFB_TMEM_ST_32(tmem_s + c * 32, sm);
              tc_wait_st();
            }
          }
          uint32_t s0[32], s1[32], s2[32], s3[32];
          XFB_TMEM_LD_32(tmem_s, s0);
          XFB_TMEM_LD_32(tmem_s + 32, s1);
          XFB_TMEM_LD_32(tmem_s + 64, s2);
          XFB_TMEM_LD_32(tmem_s + 96, s3);
          XFB_TMEM_WAIT_LD_32(s0);
          XFB_TMEM_WAIT_LD_32(s1);
          XFB_TMEM_WAIT_LD_32(s2);
          XFB_TMEM_WAIT_LD_32(s3);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar->s_empty[buf]);
          float mx = fmaxf(chunk_max(reinterpret_cast<float*>(s0)), chunk_max(reinterpret_cast<float*>(s1)));
          mx = fmaxf(mx, fmaxf(chunk_max(reinterpret_cast<float*>(s2)), chunk_max(reinterpret_cast<float*>(s3))));
          const float ms = mx * a.scale_log2;  // scale > 0
          // the previous product of the tile has to be through: P_t is free again, O_t quiescent
          if (!mbar_wait(&bar->pv_done[t], (cnt & 1) ^ 1, abort_flag, budget)) {
            code = 59 + t;
            break;
          }
          tc_fence_after();
          if (__any_sync(0xffffffffu, ms > m_run + kRescaleThreshold)) {
            const float m_new = ms > m_run + kRescaleThreshold ? ms : m_run;
            const float alpha = m_new == m_run ? 1.f : (m_run == -INFINITY ? 0.f : fast_exp2(m_run - m_new));
            if (j > 0) {
              const uint64_t al2 = f2_pack(alpha, alpha);
#pragma unroll
              for (int c = 0; c < D / 16; ++c) {
                uint32_t o[16];
                XFB_TMEM_LD_16(tmem_o + c * 16, o);
                XFB_TMEM_WAIT_LD_16(o);
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                  float x0, x1;
                  f2_unpack(fmul2(f2_pack(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), al2), x0, x1);
                  o[i] = __float_as_uint(x0), o[i + 1] = __float_as_uint(x1);
                }
                XFB_TMEM_ST_16(tmem_o + c * 16, o);
              }
              tc_wait_st();
            }
            l_run *= alpha;
            m_run = m_new;
          }
          const float m_use = m_run == -INFINITY ? 0.f : m_run;
          const uint64_t nm2 = f2_pack(-m_use, -m_use);
          uint64_t sum2[4] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f), f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
          exp_store(s0, 0, nm2, sum2);
          exp_store(s1, 16, nm2, sum2);
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar->p_half[t]);
          exp_store(s2, 32, nm2, sum2);
          exp_store(s3, 48, nm2, sum2);
          float x0, x1, y0, y1;
          f2_unpack(fadd2(sum2[0], sum2[1]), x0, x1);
          f2_unpack(fadd2(sum2[2], sum2[3]), y0, y1);
          l_run += (x0 + x1) + (y0 + y1);
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar->p_full[t]);
        }
        // ---- the partial of the row
        if (code == 0 && !mbar_wait(&bar->pv_done[t], (cnt & 1) ^ 1, abort_flag, budget)) code = 61 + t;
        if (code == 0) {
          tc_fence_after();
          // Half of the columns at a time goes through the warp's part of the tile's Q, whose last product is through, so that the rows leave in whole
          // lines: 16-byte chunks of a row XOR-ed with the row.  (A row per thread straight to memory, 16 bytes of 32 rows a store: 2.5 us a tile.)
          constexpr int kChunks = D / 8, kRowsPer = 32 / kChunks;  // of half a row; rows of a store
          const float inv = l_run == 0.f ? 0.f : 1.f / l_run;  // (a sum of NaN stays one: NaN among visible keys is not lost)
          uint8_t* stage = smem + L::kQ + t * L::kTile + (warp & 3) * (L::kTile / 4);
          const int r_first = t * kBM + (warp & 3) * 32;  // of the block
          const int n_rows = uint32_t(sg.slot) < uint32_t(a.slots) ? min(min(sg.rows - sg.row0, a.slot_rows) - r_first, 32) : 0;
          const int64_t prow = int64_t(sg.slot) * a.slot_rows + r_first;
          float* dst = a.part_o + prow * D + (lane % kChunks) * 4;
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int col = 0; col < D / 2; col += 16) {
              uint32_t o[16];
              XFB_TMEM_LD_16(tmem_o + half * (D / 2) + col, o);
              XFB_TMEM_WAIT_LD_16(o);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(stage + lane * (2 * D) + (((col / 4 + i) ^ (lane & 7)) << 4)) =
                    make_float4(__uint_as_float(o[4 * i]) * inv, __uint_as_float(o[4 * i + 1]) * inv, __uint_as_float(o[4 * i + 2]) * inv, __uint_as_float(o[4 * i + 3]) * inv);
            }
            __syncwarp();
#pragma unroll 8
            for (int i = 0; i < 32; i += kRowsPer) {
              const int rr = i + lane / kChunks;
              if (rr < n_rows) *reinterpret_cast<float4*>(dst + rr * D + half * (D / 2)) = *reinterpret_cast<const float4*>(stage + rr * (2 * D) + (((lane % kChunks) ^ (rr & 7)) << 4));
            }
            __syncwarp();
          }
          if (lane < n_rows) a.part_lse[prow + lane] = l_run == 0.f ? -INFINITY : (m_run + log2f(l_run)) * 0.6931471805599453f;
        }
        tc_fence_before();
      }
      if (a.q_tma) {  // (whatever has gone through Q's place has left it)
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar->q_empty);
      }
      if (!segment_done()) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kPvWarp0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (a.beside && blockIdx.x == gridDim.x - 1) grid_dep_wait();
}

// ---------------------------------------------------------------------------
// Join of the partials of a row: those of its item (the segments that the CTAs had of it), then those of its own keys -- the
// chunks that the decode kernel wrote, or one partial of another operator.  kWarpsPerRow warps share a row, each takes every kWarpsPerRow-th partial, U at a
// time, and they are added up in order: the result depends on nothing but the inputs.
// ---------------------------------------------------------------------------
struct MergeArgs {
  const float* pre_o;
  const float* pre_lse;
  const GroupPlan* plan;
  const int32_t* seqstart_q;
  const int32_t* seqlen_k;
  int32_t has_prefix, groups, max_q, kv_bound, block_rows, slots, slot_rows, ctas;  // ctas: of the prefix kernel
  // own partial `s` of token b * mq + i, kv head `head`, head h of its group: own_o + s * os_s + b * os_b + i * os_i + head * os_g + h * os_h
  const float* own_o;
  const float* own_lse;
  const int32_t* own_len;  // null: own_splits partials each
  int32_t own_bound, own_chunk, own_splits, mq;
  int64_t os_s, os_b, os_i, os_g, os_h;
  int64_t ls_s, ls_b, ls_i, ls_g, ls_h;
  int32_t kv_heads, q_per_kv, total_q;
  void* out;
  float* lse;
  int64_t o_sm, o_sg, o_sh, lse_sg, lse_sh;
  int32_t out_dtype, out_vec;  // out_vec: a lane's columns are one aligned store
};

constexpr int kMergeWarps = 8;

// A row of the output: where its partials are.
struct MergeRow {
  int n_pre, n;              // partials of the prefix, of all
  int64_t pre;               // row of the first of the prefix; the next ones follow slot by slot
  int64_t own_o, own_l;
  int tok, head, h;
};
__device__ __forceinline__ GroupPlan merge_plan_of_one(const MergeArgs& a) {
  const Group grp = group_at(a, 0, a.block_rows);
  const int items = items_of(a, grp);
  const Plan plan = plan_of_one(items, grp.steps, a.ctas);
  return {0, 0, grp.steps, grp.blocks, plan.share, plan.aligned, (grp.steps + plan.share - 1) / plan.share, plan.waves * a.ctas};
}
__device__ __forceinline__ int merge_group_of(const MergeArgs& a, int tok) {
  int g = 0;  // the last group that starts at or before the token (groups without tokens have none)
  for (int n = a.groups; n > 1;) {
    const int half = n / 2;
    if (__ldcg(a.seqstart_q + g + half) <= tok) g += half, n -= half;
    else n = half;
  }
  return g;
}
__device__ __forceinline__ void merge_own(const MergeArgs& a, MergeRow& row) {  // (what the call's inputs say)
  const int b = row.tok / a.mq, qi = row.tok - b * a.mq;
  int n_own = a.own_splits;
  if (a.own_len != nullptr) n_own = min(n_own, (min(max(__ldcg(a.own_len + b), 0), a.own_bound) + a.own_chunk - 1) / a.own_chunk);
  row.n = n_own;
  row.own_o = b * a.os_b + qi * a.os_i + row.head * a.os_g + row.h * a.os_h, row.own_l = b * a.ls_b + qi * a.ls_i + row.head * a.ls_g + row.h * a.ls_h;
}
__device__ __forceinline__ void merge_prefix(const MergeArgs& a, MergeRow& row, const GroupPlan& gp, int q0) {
  row.n_pre = 0, row.pre = 0;
  const int r = (row.tok - q0) * a.q_per_kv + row.h, block = r / a.block_rows;
  if (gp.steps > 0 && r >= 0 && block < gp.blocks) {
    int item = row.head * gp.blocks + block;
    int slot = gp.base + item * gp.segs, n = gp.segs;
    if (item < gp.whole) {
      slot = item, n = 1;
    } else if (!gp.aligned) {
      item -= gp.whole;
      const int p0 = gp.base + item * gp.steps, c0 = p0 / gp.share;
      slot = gp.item_base + gp.whole + item + c0, n = (p0 + gp.steps - 1) / gp.share - c0 + 1;
    }
    row.n_pre = slot < 0 ? 0 : max(0, min(n, a.slots - slot));
    row.pre = int64_t(slot) * a.slot_rows + (r - block * a.block_rows);
  }
  row.n += row.n_pre;
}
__device__ __forceinline__ float merge_lse(const MergeArgs& a, const MergeRow& row, int s) {
  return s < row.n_pre ? a.pre_lse[row.pre + int64_t(s) * a.slot_rows] : a.own_lse[row.own_l + (s - row.n_pre) * a.ls_s];
}
// The partials s0, s0 + step, ... of a row: log-sum-exps and a lane's columns.
template <int D, int U>
struct MergeLoads {
  static constexpr int V = D / 32;
  float l[U], x[U][V];
  __device__ __forceinline__ void load(const MergeArgs& a, const MergeRow& row, int s0, int step, int lane) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * step;
      l[u] = -INFINITY;
#pragma unroll
      for (int i = 0; i < V; ++i) x[u][i] = 0.f;
      if (s < row.n) {
        l[u] = merge_lse(a, row, s);
        const float* po = (s < row.n_pre ? a.pre_o + (row.pre + int64_t(s) * a.slot_rows) * D : a.own_o + row.own_o + (s - row.n_pre) * a.os_s) + lane * V;
        if constexpr (V == 4) {
          const float4 y = *reinterpret_cast<const float4*>(po);
          x[u][0] = y.x, x[u][1] = y.y, x[u][2] = y.z, x[u][3] = y.w;
        } else {
          const float2 y = *reinterpret_cast<const float2*>(po);
          x[u][0] = y.x, x[u][1] = y.y;
        }
      }
    }
  }
  __device__ __forceinline__ void add(float mx, float (&acc)[V], float& den) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float w = l[u] != -INFINITY ? __expf(l[u] - mx) : 0.f;
      den += w;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += l[u] != -INFINITY ? w * x[u][i] : 0.f;  // (NaN goes on; a partial without a visible key counts for nothing, whatever its columns hold)
    }
  }
};
// Largest log-sum-exp of a row, by a warp: -inf if no partial has a visible key, NaN if one of them saw NaN.
__device__ __forceinline__ float merge_max(const MergeArgs& a, const MergeRow& row, int lane) {
  float mx = -INFINITY;
  for (int s = lane; s < row.n; s += 32) mx = fmax_nan(mx, merge_lse(a, row, s));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmax_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  return mx;
}
template <int V>
__device__ __forceinline__ void merge_store(const MergeArgs& a, const MergeRow& row, int lane, float mx, const float (&acc)[V], float den) {
  const float inv = den == 0.f ? 0.f : 1.f / den;
  const int64_t off = int64_t(row.tok) * a.o_sm + int64_t(row.head) * a.o_sg + int64_t(row.h) * a.o_sh + lane * V;
  if (a.out_vec) {
    if (a.out_dtype == XFB200_F32) {
      if constexpr (V == 4) *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + off) = make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
      else *reinterpret_cast<float2*>(reinterpret_cast<float*>(a.out) + off) = make_float2(acc[0] * inv, acc[1] * inv);
    } else {
      uint32_t w[V / 2];
#pragma unroll
      for (int i = 0; i < V / 2; ++i)
        w[i] = a.out_dtype == XFB200_BF16 ? pack_pair<true>(acc[2 * i] * inv, acc[2 * i + 1] * inv) : pack_pair<false>(acc[2 * i] * inv, acc[2 * i + 1] * inv);
      uint32_t* const dst = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + off);
      if constexpr (V == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
      else *dst = w[0];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float val = acc[i] * inv;
      if (a.out_dtype == XFB200_F32)
        reinterpret_cast<float*>(a.out)[off + i] = val;
      else if (a.out_dtype == XFB200_BF16)
        reinterpret_cast<__nv_bfloat16*>(a.out)[off + i] = __float2bfloat16_rn(val);
      else
        reinterpret_cast<__half*>(a.out)[off + i] = __float2half_rn(val);
    }
  }
  if (a.lse != nullptr && lane == 0) a.lse[int64_t(row.head) * a.lse_sg + int64_t(row.h) * a.lse_sh + row.tok] = den == 0.f ? -INFINITY : mx + __logf(den);
}

// Before the wait for the kernel ahead: what neither kernel ahead writes, where there is a prefix kernel: whatever wrote it had ended when the first of the call's kernels began (launch_prefix).
template <int D, int kWarpsPerRow, int U>
__global__ void __launch_bounds__(kMergeWarps * 32) shared_merge_kernel(const __grid_constant__ MergeArgs a) {
  constexpr int V = D / 32, step = kWarpsPerRow;
  __shared__ float red[kMergeWarps][D + 4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % step;
  const uint32_t gw = blockIdx.x * uint32_t(kMergeWarps / step) + warp / step;
  const bool live = gw < uint32_t(a.total_q) * a.kv_heads * a.q_per_kv;
  const uint32_t gh = gw / uint32_t(a.q_per_kv);
  MergeRow row;
  row.h = int(gw - gh * a.q_per_kv), row.tok = live ? int(gh / uint32_t(a.kv_heads)) : 0, row.head = int(gh % uint32_t(a.kv_heads));
  if (!a.has_prefix) grid_dep_wait();
  const int g = merge_group_of(a, row.tok), q0 = a.has_prefix ? __ldcg(a.seqstart_q + g) : 0;
  merge_own(a, row);
  GroupPlan gp{};
  if (a.has_prefix && a.groups == 1) gp = merge_plan_of_one(a);  // (with one group the plan is a few instructions, with more it is read behind the wait)
  grid_dep_wait();
  grid_dep_launch();
  if (a.has_prefix && a.groups > 1) gp = a.plan[g];
  merge_prefix(a, row, gp, q0);
  if (!live) row.n = 0;

  MergeLoads<D, U> now;
  now.load(a, row, part, step, lane);
  float mx = -INFINITY, acc[V], den = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  if (step == 1 && row.n <= U) {  // (all of them are here)
#pragma unroll
    for (int u = 0; u < U; ++u) mx = fmax_nan(mx, now.l[u]);
  } else {
    mx = merge_max(a, row, lane);
  }
  if (mx != -INFINITY) {
    for (int s0 = part;;) {
      now.add(mx, acc, den);
      s0 += U * step;
      if (s0 >= row.n) break;
      now.load(a, row, s0, step, lane);
    }
  }
  if constexpr (step > 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) red[warp][lane * V + i] = acc[i];
    if (lane == 0) red[warp][D] = den;
    __syncthreads();
    if (part == 0) {
#pragma unroll
      for (int w = 1; w < step; ++w) {
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += red[warp + w][lane * V + i];
        den += red[warp + w][D];
      }
    }
  }
  if (part == 0 && live) merge_store<V>(a, row, lane, mx, acc, den);
}

// ------------------------------------------------------------------ host side
template <int D, bool kBf16, int kTiles>
static int launch_prefix(const Args& a, dim3 grid, cudaStream_t st) {
  // In order, so that the kernels behind it may read beside it what it reads (the decode kernel and the lengths of the merge), or beside a kernel that was launched so.
  auto kern = shared_prefix_kernel<D, kBf16, kTiles>;
  constexpr int smem = Smem<D, kTiles>::kTotal;
  static bool configured[kMaxDevices] = {false};  // the attribute belongs to the device's context
  if (first_use_on_device(configured)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_fail("shared_prefix: cudaFuncSetAttribute", e);
  }
  const cudaError_t e = launch_ordered(kern, grid, threads(kTiles), smem, st, !a.beside, a);
  return e != cudaSuccess ? cuda_fail("shared_prefix_kernel launch", e) : XFB200_OK;
}

// Warps per row: as many as let every warp have its partials in one round of loads, while the rows' warps are resident together; latency is what a
// few rows cost, getting through CTAs what many do.  Measured, us of a call with 1 / 2 / 4 / 8 warps a row, 8 of them with eight loads each (what the rule takes in brackets; 8 kv heads
// of 128 unless said): one sequence, 8 heads on one kv head, behind 40000 keys 31.8 / 23.8 / 19.5 / 17.7 / [17.0]; 2 of 64 heads behind 65536 60.4 / 57.7 / 56.6 / [56.2] / 56.1; 4 behind 601
// 12.6 / 12.0 / [11.9] / 12.0 / 12.4; 32 behind 4096 24.9 / 24.0 / [23.7] / 27.2 / 30.1; 48 behind 5000 41.2 / [38.9] / 42.4 / 45.9 / 49.2; 128 of 64 heads behind 8192
// [149] / 155 / 167 / 186 / 201; 160 tokens of 28 heads in five groups [24.7] / 30.3 / 37.1 / 50.3 / 51.4.
template <int D>
static int launch_merge(const MergeArgs& a, int partials, cudaStream_t st) {
  const int64_t rows = int64_t(a.total_q) * a.kv_heads * a.q_per_kv, resident = int64_t(sm_count()) * 32;
  auto go = [&](void (*kern)(MergeArgs), int warps_per_row) {
    const int per_cta = kMergeWarps / warps_per_row;
    return launch_early(kern, unsigned((rows + per_cta - 1) / per_cta), kMergeWarps * 32, 0, st, a);
  };
  cudaError_t e;
  if (partials > 8 && rows * 8 <= resident)
    e = partials > 32 ? go(shared_merge_kernel<D, 8, 8>, 8) : go(shared_merge_kernel<D, 8, 4>, 8);
  else if (partials > 4 && rows * 4 <= resident)
    e = go(shared_merge_kernel<D, 4, 4>, 4);
  else if (partials > 4 && (rows * 2 <= resident || partials > 16))
    e = go(shared_merge_kernel<D, 2, 4>, 2);
  else
    e = go(shared_merge_kernel<D, 1, 4>, 1);
  return e != cudaSuccess ? cuda_fail("shared_merge_kernel launch", e) : XFB200_OK;
}

static int tiles_of(int64_t rows) { return rows <= kBM ? 1 : 2; }
static size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

// What the launch needs room for: a slot for every segment, of which there are no more than items and CTAs together, and no more than CTAs where
// segments do not cross items.  From static bounds only (a captured call may be replayed after the lengths changed).
struct Layout {
  int64_t items, ctas, slots, slot_rows, steps;  // steps: most of all items
  int tiles;
  size_t own, plan, pre_o, pre_lse, total;  // offsets in the scratch
};
static Layout layout(const xfb200_shared_prefix_params* p) {
  Layout l{};
  l.own = p->own != nullptr ? decode_partials_bytes(*p->own) : 0;
  const int64_t rows = int64_t(p->max_q) * p->q_per_kv;
  l.tiles = tiles_of(rows);
  const int64_t block = int64_t(l.tiles) * kBM, steps = (int64_t(p->kv_padding) + kBN - 1) / kBN;
  l.items = std::min<int64_t>(int64_t(p->groups) * ((rows + block - 1) / block), int64_t(p->total_q) * p->q_per_kv / block + p->groups) * p->kv_heads;
  l.steps = l.items * steps;
  l.ctas = std::min<int64_t>(sm_count(), l.steps);
  l.slots = l.steps > 0 ? l.items + l.ctas : 0, l.slot_rows = std::min(block, rows);
  l.plan = l.own;
  l.pre_o = l.plan + up256(size_t(p->groups) * sizeof(GroupPlan));
  l.pre_lse = l.pre_o + up256(size_t(l.slots) * l.slot_rows * p->head_dim * 4);
  l.total = l.pre_lse + up256(size_t(l.slots) * l.slot_rows * 4);
  return l;
}

// How the decode kernel is to run.  One tile of query rows to a CTA where two do not fit its registers (16-bit cache, head dim 128: behind 700 shared keys, 48
// sequences of 32 rows a kv head and up to 32 / 512 / 2048 keys, 8 kv heads: 32.3 / 81.3 / 208 us with two tiles, 30.9 / 49.2 / 129 with one, although the keys are then
// read twice; head dim 64, where they fit: 27.4 / 36.4 / 92.9 and 27.2 / 40.6 / 88.4).
static int32_t own_flags(const xfb200_decode_params& own) {
  return XFB200_DECODE_PARTIALS_ONLY | (own.kv_format == XFB200_KV_PLAIN && own.head_dim == 128 ? XFB200_DECODE_ONE_TILE : 0);
}

// How many SMs the prefix kernel takes; the decode kernel, launched behind it, starts on the others and follows on these.  What a small model of the two says
// is over first.  A CTA of the prefix kernel costs 8 us and 1.3 us a step with one tile of rows, 1.6 with two (head dim 64: 1.1, 1.3), a step
// of one tile no less than its bytes at its share of the memory's rate; a decode CTA 4 us (two tiles of rows: 8) and its keys at 55 GB/s or its share,
// of the bounds' three quarters (lengths are not known here).  Decode CTAs that find no free SM start when the first are through; where they come
// in several waves, which share the memory with the prefix kernel, that one has to be over in the first half.
// Measured, us by SMs of the prefix kernel (head dim 128; the rule's choice last): 32 sequences behind 4096 keys 148 / 80 / 40 / 24 / 32: 29.9 / 26.4 / 24.1 / 24.8 / 23.3;
// 48 behind 5000 148 / 64 / 32 / 24 / 48: 55.2 / 49.8 / 38.8 / 44.7 / 38.9; 128 of 64 heads behind 8192, paged, 148 / 64 / 48 / 24 / 32: 166.8 / 156.2 / 151.0 / 178.8 / 149.3; 16 of 64
// heads behind 131072 96 / 148 / 128: 119.2 / 105.1 / 102.0.
static int prefix_ctas(const Layout& l, int head_dim, int groups, const xfb200_decode_params& own_) {
  xfb200_decode_params own = own_;
  own.flags = own_flags(own);
  const int sms = sm_count();
  const double step = l.tiles == 2 ? (head_dim == 64 ? 1.3 : 1.6) : (head_dim == 64 ? 1.1 : 1.3), step_us_per_cta = kBN * head_dim * 4.0 / 6.4e6;
  int64_t heads = 1;
  const int rows = own.mq * own.q_per_kv;
  const int64_t d = decode_grid(own, &heads);
  const double row_bytes = own.kv_format == XFB200_KV_PLAIN ? 2.0 * own.head_dim : own.kv_format == XFB200_KV_FP8_ROWWISE ? own.head_dim + 4.0 : own.head_dim / 2.0 + 4.0;
  const double gbs = std::min(55.0, 6400.0 / double(std::min<int64_t>(d, sms)));
  const double t_c = (rows > 16 && !(own.flags & XFB200_DECODE_ONE_TILE) ? 8.0 : 4.0) + 0.75 * 2.0 * row_bytes * double(heads) * decode_chunk_tokens(own.kv_padding, own.split_k) / (gbs * 1e3);
  int best = int(l.ctas);
  double best_us = 1e30;
  auto over = [&](int64_t n, int64_t k) {  // n CTAs of k steps
    const double t_p = 8.0 + double(k) * std::max(step, l.tiles == 1 ? double(n) * step_us_per_cta : 0.0);
    const int64_t excess = d - (sms - n);
    double t_d = 2.0 + t_c;
    if (excess > 0) t_d = std::max((double(d) * t_c + double(n) * t_p) / double(sms) + 2.0, std::min(t_p, 2.0 + (0.3 + 0.9 * double(excess) / double(d)) * t_c) + t_c);
    return std::max(d > sms ? 1.7 * t_p : t_p, t_d);
  };
  double margin = 1.0;
  if (groups == 1 && l.items <= l.ctas) {  // items cut evenly, if that is about as good
    margin = 0.98;
    const int64_t steps = l.steps / l.items;
    for (int64_t c = std::min(l.ctas / l.items, steps); c >= 1; --c) {
      const int64_t k = (steps + c - 1) / c, n = l.items * ((steps + k - 1) / k);
      const double us = over(n, k);
      if (us < best_us) best_us = us, best = int(n);
    }
  }
  const double even_us = best_us;
  for (int64_t k = (l.steps + l.ctas - 1) / l.ctas;; k = std::max(k + 1, k * 9 / 8)) {
    const int64_t n = (l.steps + k - 1) / k;
    const double us = over(n, k);
    if (us < best_us && us < margin * even_us) best_us = us, best = int(n);
    if (n <= 8 || double(k) * step > 1.5 * best_us) break;
  }
  return best;
}

}  // namespace spx
}  // namespace xfb

// Chunks per sequence for the own keys: what the decode kernel would have, or chunks of 640 tokens where these fill the machine twice -- beside the prefix kernel
// SMs come free one by one, and large CTAs would leave a long tail.  (128 sequences of up to 2056 keys behind 8192, 48 SMs for the prefix: in 2 / 3 / 4 /
// 6 chunks 165.5 / 155.4 / 150.2 / 156.9 us.)
extern "C" int32_t xfb200_shared_prefix_split_k(int32_t batch, int64_t kv_bound, int32_t kv_heads, int32_t rows, int32_t row_bytes, int32_t quantised) {
  using namespace xfb;
  const int32_t alone = xfb200_decode_split_k(batch, kv_bound, kv_heads, rows, row_bytes, quantised);
  if (batch < 1 || kv_bound < 1 || kv_heads < 1) return alone;
  int heads = 8;  // of a CTA
  while (kv_heads % heads) heads >>= 1;
  const int64_t fine = std::min<int64_t>((kv_bound + 639) / 640, 1024), blocks = kv_heads / heads;
  return batch * blocks * fine >= 2 * sm_count() ? std::max(alone, int32_t(fine)) : alone;
}

extern "C" size_t xfb200_shared_prefix_scratch_bytes(const xfb200_shared_prefix_params* p) {
  if (p == nullptr || p->groups < 1 || p->kv_heads < 1 || p->total_q < 0 || p->max_q < 0 || p->q_per_kv < 1 || p->head_dim < 1 || p->kv_padding < 0) return 0;
  return xfb::spx::layout(p).total;
}

extern "C" int xfb200_shared_prefix_forward(const xfb200_shared_prefix_params* p, void* stream) {
  using namespace xfb;
  using namespace xfb::spx;
  if (p == nullptr) return set_error(XFB200_E_INVALID, "shared_prefix: null params");
  if (p->groups < 1 || p->max_q < 0 || p->total_q < 0 || p->kv_heads < 1 || p->q_per_kv < 1 || p->kv_padding < 0)
    return set_error(XFB200_E_INVALID, "shared_prefix: bad extents");
  if (p->total_q == 0) return XFB200_OK;
  if (p->head_dim != 64 && p->head_dim != 128) return set_error(XFB200_E_UNSUPPORTED, "shared_prefix: head_dim %d not in {64, 128}", p->head_dim);
  if (p->dtype != XFB200_BF16 && p->dtype != XFB200_F16) return set_error(XFB200_E_INVALID, "shared_prefix: dtype must be bf16 or f16");
  if (p->out_dtype != XFB200_BF16 && p->out_dtype != XFB200_F16 && p->out_dtype != XFB200_F32) return set_error(XFB200_E_INVALID, "shared_prefix: bad out_dtype %d", p->out_dtype);
  if (!(p->scale > 0.f)) return set_error(XFB200_E_UNSUPPORTED, "shared_prefix: scale must be positive");
  const bool prefix = p->kv_padding > 0 && p->max_q > 0;
  if (p->q == nullptr || p->out == nullptr || p->seqstart_q == nullptr || p->seqlen_k == nullptr || (prefix && (p->k == nullptr || p->v == nullptr)))
    return set_error(XFB200_E_INVALID, "shared_prefix: null tensor pointer");
  if ((p->own != nullptr) == (p->own_out != nullptr)) return set_error(XFB200_E_INVALID, "shared_prefix: the own keys come as parameters of the decode kernel or as one partial per row");
  if (p->own_out != nullptr && ((reinterpret_cast<uintptr_t>(p->own_out) & 15) || p->own_stride_m % 4 || p->own_stride_g % 4 || p->own_stride_h % 4))
    return set_error(XFB200_E_INVALID, "shared_prefix: rows of the own partial must be 16-byte aligned");
  if (p->own_beside < 0 || p->own_beside > 1) return set_error(XFB200_E_INVALID, "shared_prefix: own_beside %d", p->own_beside);
  if (p->own_out != nullptr && p->own_lse == nullptr) return set_error(XFB200_E_INVALID, "shared_prefix: a partial without its log-sum-exp");
  if (p->scratch == nullptr || (reinterpret_cast<uintptr_t>(p->scratch) & 255)) return set_error(XFB200_E_INVALID, "shared_prefix: scratch must be given and 256-byte aligned");
  if (p->block_tables != nullptr && (p->page_size < 1 || p->block_table_stride < 0)) return set_error(XFB200_E_INVALID, "shared_prefix: page_size %d with a page table", p->page_size);
  if (p->block_tables != nullptr && p->page_size % 8) return set_error(XFB200_E_UNSUPPORTED, "shared_prefix: pages of %d tokens (a multiple of 8)", p->page_size);
  if (prefix && (p->kv_rows < 1 || p->kv_rows > 0x7fffff00)) return set_error(XFB200_E_INVALID, "shared_prefix: kv_rows %lld", (long long)p->kv_rows);
  const int64_t strides[] = {p->q_stride_m, p->q_stride_g, p->q_stride_h, p->k_stride_m, p->k_stride_g, p->v_stride_m, p->v_stride_g};
  for (int64_t s : strides)
    if (s % 8) return set_error(XFB200_E_INVALID, "shared_prefix: rows of q and of the prefix must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v)) & 15)
    return set_error(XFB200_E_INVALID, "shared_prefix: q and the prefix must be 16-byte aligned");
  if (p->own != nullptr && (p->own->kv_heads != p->kv_heads || p->own->q_per_kv != p->q_per_kv || p->own->head_dim != p->head_dim ||
                            int64_t(p->own->batch) * p->own->mq != p->total_q || p->own->window_size != 0))
    return set_error(XFB200_E_INVALID, "shared_prefix: the own keys' parameters do not belong to these queries");
  if (p->own != nullptr && (p->own->batch < 1 || p->own->mq < 1 || p->own->split_k < 1 || p->own->split_k > 1024 || p->own->kv_padding < 1))  // (before anything is worked out from them)
    return set_error(XFB200_E_INVALID, "shared_prefix: bad extents of the own keys");
  if (int64_t(p->total_q) * p->q_per_kv * p->kv_heads > 0x3fffffff) return set_error(XFB200_E_UNSUPPORTED, "shared_prefix: too many query rows");

  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Layout l = layout(p);
  if (l.steps > 0x3fffffff || l.slots > 0x3fffffff) return set_error(XFB200_E_UNSUPPORTED, "shared_prefix: %lld steps in all", (long long)l.steps);
  uint8_t* scratch = static_cast<uint8_t*>(p->scratch);
  MergeArgs m{};
  m.seqstart_q = p->seqstart_q, m.groups = p->groups;
  m.plan = reinterpret_cast<const GroupPlan*>(scratch + l.plan);
  m.has_prefix = prefix, m.seqlen_k = p->seqlen_k, m.max_q = p->max_q, m.kv_bound = p->kv_padding;
  m.ctas = p->own != nullptr && l.ctas > 0 ? prefix_ctas(l, p->head_dim, p->groups, *p->own) : int32_t(l.ctas);
  m.block_rows = l.tiles * kBM, m.slots = int32_t(l.slots), m.slot_rows = int32_t(l.slot_rows);
  m.kv_heads = p->kv_heads, m.q_per_kv = p->q_per_kv, m.total_q = p->total_q;
  m.out = p->out, m.lse = p->lse, m.out_dtype = p->out_dtype;
  {
    const int cols = p->head_dim / 32, bytes = cols * (p->out_dtype == XFB200_F32 ? 4 : 2);
    m.out_vec = reinterpret_cast<uintptr_t>(p->out) % bytes == 0 && p->o_stride_m % cols == 0 && p->o_stride_g % cols == 0 && p->o_stride_h % cols == 0;
  }
  m.o_sm = p->o_stride_m, m.o_sg = p->o_stride_g, m.o_sh = p->o_stride_h, m.lse_sg = p->lse_stride_g, m.lse_sh = p->lse_stride_h;
  m.pre_o = reinterpret_cast<const float*>(scratch + l.pre_o), m.pre_lse = reinterpret_cast<const float*>(scratch + l.pre_lse);

  if (prefix) {
    Args a{};
    EncodeTiledFn enc = encode_tiled_fn();
    if (enc == nullptr) return set_error(XFB200_E_CUDA, "shared_prefix: cuTensorMapEncodeTiled is not available from this driver");
    a.box_tok = kBN;
    if (p->block_tables != nullptr)
      while (p->page_size % a.box_tok) a.box_tok >>= 1;
    auto map = [&](CUtensorMap* tm, const void* base, int64_t sm, int64_t sg, int32_t* step) -> int {
      const bool one = p->kv_heads == 1 || sg == 0;
      *step = one ? 0 : 1;
      const cuuint64_t dims[3] = {cuuint64_t(p->head_dim), cuuint64_t(p->kv_rows), cuuint64_t(one ? 1 : p->kv_heads)};
      const cuuint64_t str[2] = {cuuint64_t(p->kv_rows == 1 ? p->head_dim : sm) * 2, cuuint64_t(one ? p->head_dim : sg) * 2};
      const cuuint32_t box[3] = {64, cuuint32_t(a.box_tok), 1}, estr[3] = {1, 1, 1};
      const CUresult r = enc(tm, p->dtype == XFB200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, str, box, estr,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
      return r != CUDA_SUCCESS ? set_error(XFB200_E_INVALID, "shared_prefix: a tensor map cannot describe the prefix (CUresult %d)", int(r)) : XFB200_OK;
    };
    int rc = map(&a.tm_k, p->k, p->k_stride_m, p->k_stride_g, &a.k_heads_step);
    if (rc == XFB200_OK) rc = map(&a.tm_v, p->v, p->v_stride_m, p->v_stride_g, &a.v_heads_step);
    if (rc != XFB200_OK) return rc;
    // Q by tiled copies where 128 rows are whole tokens (4 sequences of 4 rows a kv head behind 601 keys, with stores by the softmax warps and so: 11.5 / 11.0 us; 1753
    // tokens behind 16384: 414 / 411)
    if (p->q_per_kv <= kBM && (p->q_per_kv & (p->q_per_kv - 1)) == 0) {
      const int64_t ext[3] = {p->q_per_kv, p->kv_heads, p->total_q}, st[3] = {p->q_stride_h, p->q_stride_g, p->q_stride_m};
      cuuint64_t dims[4] = {cuuint64_t(p->head_dim)}, str[3];
      bool ok = true;
      for (int i = 0; i < 3; ++i) ok = ok && (ext[i] == 1 || st[i] > 0), dims[i + 1] = cuuint64_t(ext[i]), str[i] = cuuint64_t(ext[i] == 1 ? p->head_dim : st[i]) * 2;
      const cuuint32_t box[4] = {64, cuuint32_t(p->q_per_kv), 1, cuuint32_t(kBM / p->q_per_kv)}, estr[4] = {1, 1, 1, 1};
      a.q_tma = ok && enc(&a.tm_q, p->dtype == XFB200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(p->q), dims, str, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    }
    int32_t* words = device_words();
    if (words == nullptr) return set_error(XFB200_E_CUDA, "shared_prefix: cannot resolve the device status word");
    a.status = words + kWordPrefillStatus;
    a.q = p->q, a.part_o = const_cast<float*>(m.pre_o), a.part_lse = const_cast<float*>(m.pre_lse);
    a.seqstart_q = p->seqstart_q, a.seqlen_k = p->seqlen_k, a.block_tables = p->block_tables, a.bt_stride = p->block_table_stride, a.kv_rows = p->kv_rows;
    a.q_sm = p->q_stride_m, a.q_sg = p->q_stride_g, a.q_sh = p->q_stride_h;
    a.groups = p->groups, a.kv_heads = p->kv_heads, a.q_per_kv = p->q_per_kv, a.total_q = p->total_q;
    a.max_q = p->max_q, a.kv_bound = p->kv_padding, a.page_size = p->page_size;
    a.plan = const_cast<GroupPlan*>(m.plan), a.slots = m.slots, a.slot_rows = m.slot_rows;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    a.wait_budget = wait_units(p->wait_budget_kcycles > 0 ? 1000LL * p->wait_budget_kcycles : kWaitBudgetCycles);
    a.debug_flags = p->debug_flags;
    a.beside = p->own_out != nullptr && p->own_beside != 0;
    dim3 grid(unsigned(m.ctas), 1, 1);
    const bool bf16 = p->dtype == XFB200_BF16;
    if (p->head_dim == 128)
      rc = l.tiles == 1 ? (bf16 ? launch_prefix<128, true, 1>(a, grid, st) : launch_prefix<128, false, 1>(a, grid, st))
                      : (bf16 ? launch_prefix<128, true, 2>(a, grid, st) : launch_prefix<128, false, 2>(a, grid, st));
    else
      rc = l.tiles == 1 ? (bf16 ? launch_prefix<64, true, 1>(a, grid, st) : launch_prefix<64, false, 1>(a, grid, st))
                      : (bf16 ? launch_prefix<64, true, 2>(a, grid, st) : launch_prefix<64, false, 2>(a, grid, st));
    if (rc != XFB200_OK) return rc;
  }
  if (p->own != nullptr) {
    xfb200_decode_params own = *p->own;
    own.q = p->q, own.out = p->out, own.lse = nullptr, own.scratch = scratch;
    own.q_stride_m = p->q_stride_m, own.q_stride_g = p->q_stride_g, own.q_stride_h = p->q_stride_h;
    own.dtype = p->dtype, own.scale = p->scale, own.out_dtype = p->out_dtype;
    own.flags = own_flags(own) | (prefix ? XFB200_DECODE_BESIDE : 0);
    const int rc = xfb200_decode_forward(&own, stream);
    if (rc != XFB200_OK) return rc;
    const int64_t R = int64_t(own.mq) * own.q_per_kv, per_split = own.kv_heads * R;
    m.own_o = reinterpret_cast<const float*>(scratch), m.own_lse = reinterpret_cast<const float*>(scratch + decode_partials_lse_offset(own));
    m.own_len = own.seqlen_k, m.own_bound = own.kv_padding, m.own_chunk = decode_chunk_tokens(own.kv_padding, own.split_k), m.mq = own.mq;
    m.own_splits = std::min(own.split_k, (own.kv_padding + m.own_chunk - 1) / m.own_chunk);
    m.ls_s = per_split, m.ls_b = own.split_k * per_split, m.ls_i = own.q_per_kv, m.ls_g = R, m.ls_h = 1;
    m.os_s = m.ls_s * own.head_dim, m.os_b = m.ls_b * own.head_dim, m.os_i = m.ls_i * own.head_dim, m.os_g = m.ls_g * own.head_dim, m.os_h = own.head_dim;
  } else {
    m.own_o = p->own_out, m.own_lse = p->own_lse, m.own_splits = 1, m.mq = 1;
    m.os_b = p->own_stride_m, m.os_g = p->own_stride_g, m.os_h = p->own_stride_h;
    m.ls_b = 1, m.ls_g = p->own_lse_stride_g, m.ls_h = p->own_lse_stride_h;
  }
  // partials of a row, as far as the bounds tell
  const int64_t steps = (int64_t(p->kv_padding) + kBN - 1) / kBN, cut = l.items > 0 ? m.ctas / l.items + (m.ctas < l.items) : 0;
  const int most = int(std::min(cut, steps)) + m.own_splits;
  return p->head_dim == 128 ? launch_merge<128>(m, most, st) : launch_merge<64>(m, most, st);
}
