// Chunked-prefill paged attention on the 5th-generation tensor cores (tcgen05 + TMEM).
//
// A work record is a run of up to 2 x (128/G) consecutive rows of one sequence.  The G query heads of
// one KV head of those rows are packed into TWO query tiles of 128 rows each (tile t = rows
// [t*128/G, (t+1)*128/G) of the record); both tiles attend to the KV range [kv_begin, kv_end) of the pool
// (prefix + the rows themselves, causal inside the chunk), so every K/V tile is fetched once for 256
// packed rows.  Q.K^T (128 x T x d) and P.V (128 x d x T) run as tcgen05.mma.kind::f16 with fp32
// accumulators in tensor memory.  The description below is head_dim 128 (KV tiles of T = 128 tokens);
// head_dim 64 is the same with 64-column accumulators, and head_dim 256, whose two 256-column accumulators
// would not fit beside the scores, runs ONE query tile per CTA (the record's two tiles go to two CTAs)
// against KV tiles of 64 tokens, so that two K and three V stages still fit in shared memory; there the two
// score buffers alternate between consecutive KV tiles and Q.K^T runs two tiles ahead of P.V:
//
//   TMEM (512 columns)   S0 | S1 | O0 | O1, 128 columns each; P_t (bf16, 64 columns) overwrites the lower
//                        half of S_t and is the A operand of P_t.V straight from tensor memory
//   warps 0-3 / 4-7      softmax of query tile 0 / 1: thread = one packed row = one TMEM lane, all 128
//                        columns, so the row maximum and the row sum need no exchange with anybody.
//                        S comes in with tcgen05.ld, P (rounded to bf16, the reference's boundary) goes
//                        back with tcgen05.st; O is rescaled in TMEM only when the running maximum moved
//                        by more than 2^8; at the end the same thread normalises its O row and stores it
//                        to every destination
//   warps 8-11           loaders (8-9 K, 10-11 V) of 128-token tiles: whole, slot-contiguous pages by TMA
//                        (cp.async.bulk.tensor 2-D boxes, 128-byte swizzle, no multicast), anything else
//                        row by row with 16-byte cp.async; two K stages, three V stages
//   warp 12              one thread issues the MMAs in the order  P0.V(j), Q0.K(j+1), P1.V(j), Q1.K(j+1):
//                        while one tile's softmax runs, the tensor pipe works on the other tile
//
// While one tile's softmax runs, the tensor pipe has the other tile's two products to do.  The softmax
// arithmetic is packed (fma.f32x2 / add.f32x2, three-input maxima) and the uncommon cases (softcap, tiles
// that need masking) rewrite S in tensor memory in a short loop first, so the common path stays small:
// the instruction cache is the first thing this kernel ran out of when every case was unrolled in place.
// Every mbarrier wait is bounded: on expiry the CTA raises GK_DEV_WAIT_EXPIRED, drains its copies,
// frees its TMEM and returns.
#include "tc_common.cuh"

#include <string.h>
#include <math_constants.h>

namespace gk {
namespace {

constexpr int kRows = 128;             // packed query rows per tile = lanes of tensor memory
constexpr int kKStages = 2, kVStages = 3;
constexpr int kSoftmaxThreads = 256, kLoaderThreads = 64, kThreads = 512;   // loaders: 64 threads for K, 64 for V
constexpr int kLaunchRegs = 128;     // what __launch_bounds__(512, 1) lets ptxas allocate per thread
constexpr int kSoftmaxRegs = 184, kLoaderRegs = 80, kIssueRegs = 64;
static_assert(kSoftmaxThreads * kSoftmaxRegs + 128 * kLoaderRegs + 128 * kIssueRegs <= kThreads * kLaunchRegs,
              "register budgets exceed the pool the launch allocates");

// Shapes that follow from head_dim D.  Operand tiles are stored as D/64 panels of [rows x 128 bytes] with the
// 128-byte swizzle; a query tile has 128 rows, a K or V tile kKv rows.
template <int D>
struct Geo {
  static_assert(D == 64 || D == 128 || D == 256, "head_dim");
  static constexpr int kKv = D == 256 ? 64 : 128;          // KV tokens per tile
  static constexpr int kTiles = D == 256 ? 1 : 2;          // query tiles per CTA
  static constexpr int kPanels = D / 64, kChunks = D / 8;  // 128-byte panels, 16-byte chunks per row
  static constexpr int kQPanelBytes = kRows * 128, kQTileBytes = kPanels * kQPanelBytes;
  static constexpr int kKvPanelBytes = kKv * 128, kKvTileBytes = kPanels * kKvPanelBytes;
  static constexpr int kSmemBytes = kTiles * kQTileBytes + (kKStages + kVStages) * kKvTileBytes + 3072;
  // kind::f16 instruction descriptors: fp32 accumulate, bf16 x bf16, M = 128; N = kKv (A, B K-major) for the
  // scores, N = D with B (= V) MN-major for the second product.
  static constexpr uint32_t kIdescQK = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kKv >> 3) << 17) | (8u << 24);
  static constexpr uint32_t kIdescPV = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | (8u << 24);
};
static_assert(Geo<128>::kSmemBytes <= 227 * 1024 && Geo<256>::kSmemBytes <= 227 * 1024, "shared memory of an SM");
constexpr float kLog2e = 1.4426950408889634f;

struct PrefillParams {
  const __nv_bfloat16* q;
  const __nv_bfloat16* pool_k;
  const __nv_bfloat16* pool_v;
  const int32_t* table;
  const int32_t* table_rows;
  const int32_t* work;
  __nv_bfloat16* out[GK_MAX_OUTPUTS];   // every destination receives the same rows (peers under TP)
  int32_t* status;
  int64_t q_stride, out_stride, slots, table_stride, entry_stride;
  float scale, softcap;
  int window, page_shift, q_heads, kv_heads, group;
  int tma_rows;          // rows of a TMA box, 0 = TMA path off
  int n_out;
  // read by the biased and the shared forms only (template arguments), the first two may be null:
  const float* slopes;          // [q_heads]: the score of key j gets -slope * |position - j|
  const int32_t* row_limits;    // [rows]: last key a row sees, at or behind its position (two-way prefix)
  const int4* list;             // shared form: {row, position, first entry, entries between two parts} per listed row
  float* part_ml;               // shared form: (m in log2 units, l) and un-normalised O of every entry
  float* part_o;
};

struct Shared {
  uint64_t k_full[kKStages + 1], k_free[kKStages + 1], v_full[kVStages], v_free[kVStages];
  uint64_t s_full[2], p_full[2], pv_done[2];
  uint32_t tmem_base;
  int abort;
};

// Byte offset of 16-byte chunk c of row r inside a tile whose panels are panel_bytes apart.
__device__ __forceinline__ uint32_t tile_off(int r, int c, int panel_bytes) {
  return (c >> 3) * panel_bytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// The MMAs take each 64-bit shared-memory descriptor as its two halves: the upper half (strides, swizzle mode)
// is the same for every tile of one operand kind, the lower half is the address field plus the
// leading-dimension stride, so stepping through a tile or a ring is a 32-bit add.  The second form reads its
// A operand (P, bf16, two per 32-bit column) from tensor memory.
__device__ __forceinline__ void umma_bf16_ss_split(uint32_t tmem_d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                                   uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 da, db;\nsetp.ne.b32 p, %6, 0;\nmov.b64 da, {%1, %2};\nmov.b64 db, {%3, %4};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n}\n" ::"r"(tmem_d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_bf16_ts_split(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                                   uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 db;\nsetp.ne.b32 p, %5, 0;\nmov.b64 db, {%2, %3};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st16_nowait(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// BIASED: a distance bias and row limits.
// FORM: kRowsForm is the kernel described above.  The shared forms attend to keys that several sequences have in common:
// the rows of a record are listed, every listed row sees all of the record's keys but for its window, and the state
// (m, l, O) is left for the merge instead of a normalised row.  A record is {first listed row, n_rows, part, table_row,
// kv_begin, kv_end, largest position, 0}.  kWideForm takes two query tiles like kRowsForm.  kNarrowForm (head_dim 64 and
// 128) takes one: its even KV tiles are the work of softmax warps 0-3, S0 and O0, its odd ones of warps 4-7, S1 and O1, so
// the tensor pipe still has two independent chains although a K/V tile is read for one query tile only, Q.K^T runs two KV
// tiles ahead, and the room of the second query tile is a third K stage; the two chains' states are merged through shared
// memory at the end.
// CAP: the scores are capped (the biased and the shared kernels are built with and without: the common path of one that has
// the cap's code beside it ran 5 % slower).  The plain kernel decides at run time.
constexpr int kRowsForm = 0, kWideForm = 1, kNarrowForm = 2;
template <int D, bool BIASED, int FORM, bool CAP>
__global__ void __launch_bounds__(kThreads, 1) paged_prefill_tc_kernel(const PrefillParams p,
                                                                       const __grid_constant__ CUtensorMap map_k,
                                                                       const __grid_constant__ CUtensorMap map_v) {
  using G_ = Geo<D>;
  constexpr int kKv = G_::kKv, kTiles = G_::kTiles, kChunks = G_::kChunks;
  constexpr int kQPanelBytes = G_::kQPanelBytes, kQTileBytes = G_::kQTileBytes;
  constexpr int kKvPanelBytes = G_::kKvPanelBytes, kKvTileBytes = G_::kKvTileBytes;
  constexpr int kScoreChunks = kKv / 32;                 // 32-column pieces of a row of S
  constexpr bool SHARED = FORM != kRowsForm, NARROW = FORM == kNarrowForm;
  static_assert(!NARROW || kTiles == 2, "the narrow form needs room for two accumulators in tensor memory");
  constexpr int kQTiles = NARROW ? 1 : kTiles, kKRing = NARROW ? kKStages + 1 : kKStages;
  extern __shared__ __align__(1024) uint8_t tiles[];     // swizzle atoms need 1 KiB alignment
  uint8_t* s_q = tiles;                                  // the query tiles
  uint8_t* s_k = s_q + kQTiles * kQTileBytes;            // K stages
  uint8_t* s_v = s_k + kKRing * kKvTileBytes;            // V stages
  Shared* sh = reinterpret_cast<Shared*>(s_v + kVStages * kKvTileBytes);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (smem_u32(tiles) & 1023) {                          // cannot build valid descriptors: report, leave
    if (tid == 0 && p.status) atomicOr(p.status, (int)GK_DEV_WAIT_EXPIRED);
    return;
  }
  // With one query tile per CTA the record's two tiles go to two consecutive CTAs.
  const int unit = kTiles == 2 ? blockIdx.x : blockIdx.x >> 1, half = kTiles == 2 ? 0 : blockIdx.x & 1;
  const int item = unit / p.kv_heads, head = unit - item * p.kv_heads;
  const int4 w0 = __ldg(reinterpret_cast<const int4*>(p.work) + 2 * item);
  const int4 w1 = __ldg(reinterpret_cast<const int4*>(p.work) + 2 * item + 1);
  const int G = p.group;
  const int tile_rows = kRows / G;                          // rows of the record per query tile
  // last key that row `row`, at position `pos`, sees
  auto last_seen = [&](int row, int pos) { return BIASED && p.row_limits ? __ldg(p.row_limits + row) : pos; };
  int first_row = w0.x, n_rows = w0.y, first_pos = w0.z, kv_begin = w1.x, kv_end = w1.y;
  const int table_row = w0.w;
  if (kTiles == 1) {                                        // this CTA's tile of the record, as a record of its own
    const int skip = half * tile_rows;
    n_rows = min(n_rows - skip, tile_rows);
    if (n_rows <= 0) return;                                // the whole CTA: nothing is allocated yet
    first_row += skip;
    if (!SHARED) {
      first_pos += skip;
      kv_end = min(kv_end, last_seen(first_row + n_rows - 1, first_pos + n_rows - 1) + 1);   // causal: nothing after this tile's last row
      if (p.window > 0) kv_begin = max(kv_begin, first_pos - p.window + 1);
    }
  }
  const int rows0 = min(n_rows, tile_rows), rows1 = NARROW ? rows0 : n_rows - rows0;
  const int tile_step = NARROW ? 0 : tile_rows;             // rows between the two tiles (chains)
  // The first record of a shared prefix may begin inside a tile (the first key that any of its rows' windows shows): its
  // tiles stay on the pool's boxes, and what lies in front of it is zeros like what lies behind kv_end.
  const int kv_seen = kv_begin;
  if (SHARED) kv_begin = kv_begin / kKv * kKv;
  // KV tiles each query tile needs: tile 0 stops at its own last row (causal), tile 1 at the record's end
  const int nt1_all = (kv_end - kv_begin + kKv - 1) / kKv;
  const int nt0 = NARROW ? (nt1_all + 1) / 2 : SHARED ? nt1_all : min(nt1_all, (last_seen(first_row + rows0 - 1, first_pos + rows0 - 1) + 1 - kv_begin + kKv - 1) / kKv);
  const int nt1 = NARROW ? nt1_all / 2 : rows1 > 0 ? nt1_all : 0;
  const int n_tiles = NARROW ? nt1_all : max(nt0, nt1);
  // Under a distance bias the nearest keys weigh most: the biased kernel walks the KV range backwards, so that the running
  // maximum is there after the first tile.  Forwards it grew with every tile, and each time O was rescaled in tensor
  // memory behind a wait for the product before (12 % of the launch).  A query tile whose range ends earlier then starts
  // later: its first KV tile is number `head0`.
  const int head0 = BIASED && !NARROW ? n_tiles - nt0 : 0;
  auto tile_at = [&](int j) { return kv_begin + (BIASED ? n_tiles - 1 - j : j) * kKv; };

  if (tid == 0) {
    for (int i = 0; i < kKRing; ++i) {
      bar_init(&sh->k_full[i], kLoaderThreads);
      bar_init(&sh->k_free[i], 1);
    }
    for (int i = 0; i < kVStages; ++i) {
      bar_init(&sh->v_full[i], kLoaderThreads);
      bar_init(&sh->v_free[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(&sh->s_full[i], 1);
      bar_init(&sh->p_full[i], 4);      // one arrival per softmax warp of the tile
      bar_init(&sh->pv_done[i], 1);
    }
    sh->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&sh->tmem_base)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
  }
  // The attention kernel behind the shared forms is released once the kernel before them has completed: it reads the queries
  // and the pool without waiting for this one.
  if (SHARED) asm volatile("griddepcontrol.wait;\ngriddepcontrol.launch_dependents;\n" ::: "memory");
  tc_fence_before();
  __syncthreads();                                       // barriers and the TMEM allocation are in place
  tc_fence_after();
  const bool is_loader = warp >= 8 && warp < 12;
  if (!is_loader) {
    // Q tiles: packed row pr of tile t = (row t*tile_rows + pr / G, query head pr % G) of this KV head; unused rows
    // are zero.  The loader warps do not take part: their first K/V tiles are already on the way meanwhile.
    // Warps 0-7 take kQTiles * 16 rows each: a lane finds the place of one row (one division, one look at the list), then
    // the warp copies the rows in turn, 512 bytes an instruction, all of them under way at once.
    if (warp < 8) {
      constexpr int kWarpRows = kQTiles * 16, kRowsAtOnce = 32 / kChunks;
      const bool q_aligned = ((reinterpret_cast<uintptr_t>(p.q) | (uintptr_t)(p.q_stride * 2)) & 15) == 0;
      int64_t place = -1;                                  // of the row warp * kWarpRows + lane, in elements of q
      {
        const int at = warp * kWarpRows + lane, t = at / kRows, pr = at & (kRows - 1), r = t * tile_rows + pr / G;
        if (lane < kWarpRows && pr < tile_rows * G && r < n_rows)
          place = (int64_t)(SHARED ? __ldg(&p.list[first_row + r].x) : first_row + r) * p.q_stride + (int64_t)(head * G + pr % G) * D;
      }
      const int c = lane & (kChunks - 1);
      auto target = [&](int at) { return s_q + (at / kRows) * kQTileBytes + tile_off(at & (kRows - 1), c, kQPanelBytes); };
      if (q_aligned) {
#pragma unroll
        for (int i = 0; i < kWarpRows; i += kRowsAtOnce) {
          const int64_t from = __shfl_sync(0xffffffffu, place, i + lane / kChunks);
          cp_async_16(smem_u32(target(warp * kWarpRows + i + lane / kChunks)), p.q + (from < 0 ? 0 : from + c * 8), from < 0 ? 0 : 16);
        }
        asm volatile("cp.async.wait_all;\n" ::: "memory");
      } else {
        // Rows that are 2-byte aligned only: the six elements of a chunk that make whole words come as words, the other two
        // (its ends, or its last two) by themselves; four chunks under way at once.  Each element loaded on its own and
        // waited for by its store made the whole call 1.2 to 1.8 times as long (16 chunks of 128 rows, 32 heads of 128: 48
        // us, now 31; rows on 16-byte boundaries 29).
        constexpr int kBatch = 4;
        static_assert(kWarpRows % (kBatch * kRowsAtOnce) == 0, "whole batches");
#pragma unroll 1
        for (int i = 0; i < kWarpRows; i += kBatch * kRowsAtOnce) {
          uint32_t w[kBatch][3], one[kBatch], last[kBatch];
          bool odd[kBatch], used[kBatch];
#pragma unroll
          for (int b = 0; b < kBatch; ++b) {
            const int64_t from = __shfl_sync(0xffffffffu, place, i + b * kRowsAtOnce + lane / kChunks);
            const unsigned short* src = reinterpret_cast<const unsigned short*>(p.q) + (from < 0 ? 0 : from + c * 8);
            used[b] = from >= 0;
            odd[b] = reinterpret_cast<uintptr_t>(src) & 2;
            const uint32_t* words = reinterpret_cast<const uint32_t*>(src + (odd[b] ? 1 : 0));
#pragma unroll
            for (int k = 0; k < 3; ++k) w[b][k] = __ldg(words + k);
            one[b] = __ldg(src + (odd[b] ? 0 : 6));
            last[b] = __ldg(src + 7);
          }
#pragma unroll
          for (int b = 0; b < kBatch; ++b) {
            uint4 v;
            v.x = odd[b] ? one[b] | w[b][0] << 16 : w[b][0];
            v.y = odd[b] ? __funnelshift_r(w[b][0], w[b][1], 16) : w[b][1];
            v.z = odd[b] ? __funnelshift_r(w[b][1], w[b][2], 16) : w[b][2];
            v.w = (odd[b] ? w[b][2] >> 16 : one[b]) | last[b] << 16;
            *reinterpret_cast<uint4*>(target(warp * kWarpRows + i + b * kRowsAtOnce + lane / kChunks)) = used[b] ? v : make_uint4(0, 0, 0, 0);
          }
        }
      }
    }
    fence_async_smem();
    asm volatile("bar.sync 1, %0;\n" ::"n"(kThreads - 128) : "memory");      // the 384 threads that filled Q
  }
  const uint32_t tmem = sh->tmem_base;
  // Completion of P.V(j).  Two query tiles: S(j + 1) of a tile is issued behind its P.V(j), so whoever has seen S(j) knows
  // of every product up to P.V(j - 1) and one barrier per tile is unambiguous.  One query tile: Q.K^T runs two KV tiles
  // ahead and seeing S(j) only tells of P.V(j - 2); a wait on the parity of P.V(j) alone would then pass while P.V(j - 1)
  // is still running, so consecutive products take turns on two barriers.
  auto pv_bar = [&](int t, int j) { return &sh->pv_done[kTiles == 2 ? t : (j & 1)]; };
  auto pv_phase = [&](int j) { return (uint32_t)((kTiles == 2 ? j : (j >> 1)) & 1); };

  // Registers move from the loader / issue warpgroups (which need few) to the softmax warpgroups.
  // setmaxnreg.inc blocks until the CTA's register pool can satisfy it, and the pool is what the
  // launch allocated (kThreads x kLaunchRegs): the budgets must fit in it or the softmax warps
  // would never start (checked at compile time and again on the host before every launch).
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kSoftmaxRegs));
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kLoaderRegs));
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kIssueRegs));
  }

  if (warp < 8) {
    // ================================ softmax of query tile t ===============================
    const int t = warp >> 2;
    const int pr = tid & 127;                                    // packed row == TMEM lane
    const int my_rows = t == 0 ? rows0 : rows1;
    const int mv = my_rows * G;                                  // packed rows of this tile in use
    const int my_tiles = t == 0 ? nt0 : nt1;
    const int tile_first_pos = first_pos + t * tile_step;
    int lim = pr < mv ? tile_first_pos + pr / G : 0x7fffffff;         // last visible key of this row
    int pos = lim;                                                     // its position
    int4 listed = make_int4(0, 0, 0, 0);
    if (SHARED) {
      if (pr < mv) listed = __ldg(p.list + first_row + t * tile_step + pr / G);
      pos = pr < mv ? listed.y : 0x7fffffff;
      lim = 0x7fffffff;
    } else if (BIASED && pr < mv) {
      lim = last_seen(first_row + t * tile_step + pr / G, pos);
    }
    // bias per token of distance, in log2 units
    const float slope = BIASED && p.slopes && pr < mv ? __ldg(p.slopes + head * G + pr % G) * kLog2e : 0.f;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_addr = tmem + 256 + t * D + lane_base;
    const bool capped = BIASED || SHARED ? CAP : p.softcap > 0.f;
    const float to_log2 = capped ? kLog2e : p.scale * kLog2e;
    const float cap_in = capped ? p.scale / p.softcap : 0.f;
    const float cap_exp = 2.f * kLog2e * cap_in, cap_log2 = p.softcap * kLog2e;     // see capped_scores
    const bool steep = BIASED && __any_sync(0xffffffffu, fabsf(slope) * 31.f > 100.f);
    float m = -CUDART_INF_F, l = 0.f;                            // m: exponent reference of this row
    bool alive = true;
    for (int j = 0; j < my_tiles && alive; ++j) {
      // Two query tiles: tile t owns score buffer t.  One query tile: the two buffers alternate between
      // consecutive KV tiles, so Q.K^T of the next tile is already there when this softmax ends.
      const int buf = kTiles == 2 ? t : (j & 1);
      const uint32_t use = kTiles == 2 ? j : (j >> 1);            // how often this buffer was filled before
      const uint32_t s_addr = tmem + buf * 128 + lane_base;       // S; P overwrites its lower half
      const uint32_t p_addr = s_addr;
      alive = __all_sync(0xffffffffu, bar_wait(&sh->s_full[buf], use & 1, &sh->abort));
      if (!alive) break;
      tc_fence_after();
      const int tok0 = tile_at(NARROW ? 2 * j + t : t == 0 ? j + head0 : j);
      const int tile_end = tok0 + kKv;
      const bool ragged = SHARED ? tile_end > kv_end || (p.window > 0 && tok0 <= w1.z - p.window)
                                 : tile_end > kv_end || tile_end > tile_first_pos + 1 ||
                                       (p.window > 0 && tok0 <= tile_first_pos + my_rows - 1 - p.window);
      const float from = BIASED ? (float)(tok0 - pos) : 0.f;      // key tok0 + e is at distance |from + e|
      // Softcap and tiles that need masking are uncommon: they first rewrite S in tensor memory (scores in
      // log2 units, masked keys at -inf), 32 columns at a time in a loop that is NOT unrolled, so that
      // the two passes below stay one short piece of code (the instruction cache is what this kernel
      // runs out of first when every variant is unrolled 128 times).
      float mult = to_log2;
      // Tiles whose scores cannot stay what they are go through an exact rewrite: a cap, slopes too steep for the estimate
      // of the maximum below, and biased rows that see keys behind them (there the bias falls again).
      const bool rewrite = BIASED || SHARED ? capped || (BIASED && p.slopes && (steep || (p.row_limits && tile_end > tile_first_pos + 1)))
                                            : capped || ragged;
      const float fast_slope = BIASED && !rewrite ? slope : 0.f;
      if (rewrite || ragged) {
        if (BIASED || SHARED) {
          // The keys a row sees are one interval: a key is in it when its distance from the first one is at most `span`.
          int low = p.window > 0 ? pos - p.window + 1 : 0, span = min(lim, kv_end - 1) - low;
          if (span < 0) {                               // no key at all: an interval in front of every tile
            low = 0x7fffffff;
            span = 0;
          }
          const int rel = tok0 - low;
          if (rewrite) {
#pragma unroll 1
            for (int c = 0; c < kScoreChunks; ++c) {
              uint32_t r[32];
              tmem_ld32(s_addr + c * 32, r);
              float big = 0.f;
#pragma unroll
              for (int e = 0; e < 32; e += 2) big = max3(big, fabsf(__uint_as_float(r[e])), fabsf(__uint_as_float(r[e + 1])));
              if (capped && __all_sync(0xffffffffu, big * cap_in <= 0.5f)) {
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                  float2 v = capped_small_scores(make_float2(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), cap_in, p.scale * kLog2e);
                  if (BIASED) {
                    v.x = fmaf(-slope, fabsf(from + (float)(c * 32 + e)), v.x);
                    v.y = fmaf(-slope, fabsf(from + (float)(c * 32 + e + 1)), v.y);
                  }
                  r[e] = __float_as_uint((unsigned)(rel + c * 32 + e) <= (unsigned)span ? v.x : -CUDART_INF_F);
                  r[e + 1] = __float_as_uint((unsigned)(rel + c * 32 + e + 1) <= (unsigned)span ? v.y : -CUDART_INF_F);
                }
              } else if (capped && p.softcap > kTightCap) {
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                  float2 v = capped_scores(make_float2(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), cap_in, p.scale * kLog2e, cap_exp, cap_log2);
                  if (BIASED) {
                    v.x = fmaf(-slope, fabsf(from + (float)(c * 32 + e)), v.x);
                    v.y = fmaf(-slope, fabsf(from + (float)(c * 32 + e + 1)), v.y);
                  }
                  r[e] = __float_as_uint((unsigned)(rel + c * 32 + e) <= (unsigned)span ? v.x : -CUDART_INF_F);
                  r[e + 1] = __float_as_uint((unsigned)(rel + c * 32 + e + 1) <= (unsigned)span ? v.y : -CUDART_INF_F);
                }
              } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  float v = __uint_as_float(r[e]);
                  v = capped ? capped_large_score(v, cap_exp, cap_log2) : v * to_log2;
                  if (BIASED) v = fmaf(-slope, fabsf(from + (float)(c * 32 + e)), v);
                  r[e] = __float_as_uint((unsigned)(rel + c * 32 + e) <= (unsigned)span ? v : -CUDART_INF_F);
                }
              }
              tmem_st32(s_addr + c * 32, r);
            }
          } else {
#pragma unroll 1
            for (int c = 0; c < kScoreChunks; ++c) {
              const int at = rel + c * 32;
              if (!__any_sync(0xffffffffu, at < 0 || at + 31 > span)) continue;      // every row of the warp sees all 32
              uint32_t r[32];
              tmem_ld32(s_addr + c * 32, r);
#pragma unroll
              for (int e = 0; e < 32; ++e) r[e] = (unsigned)(at + e) <= (unsigned)span ? r[e] : 0xff800000u;      // -infinity
              tmem_st32(s_addr + c * 32, r);
            }
          }
        } else {
#pragma unroll 1
        for (int c = 0; c < kScoreChunks; ++c) {
          uint32_t r[32];
          tmem_ld32(s_addr + c * 32, r);
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            float v = __uint_as_float(r[e]);
            if (capped) v = p.softcap * tanhf(v * cap_in);
            v *= to_log2;
            const int tok = tok0 + c * 32 + e;
            const bool seen = tok < kv_end && tok <= lim && (p.window <= 0 || tok > pos - p.window);
            r[e] = __float_as_uint(seen ? v : -CUDART_INF_F);
          }
          tmem_st32(s_addr + c * 32, r);
        }
        }
        if (rewrite) mult = 1.f;
      }
      // ---- the whole row comes in once (up to 128 registers) and stays until it has become P ----
      uint32_t sr[kScoreChunks][32];
#pragma unroll
      for (int c = 0; c < kScoreChunks; ++c) tmem_ld32_nowait(s_addr + c * 32, sr[c]);
      tmem_ld_wait();
      float mx;
      {
        float part[kScoreChunks];
#pragma unroll
        for (int c = 0; c < kScoreChunks; ++c) part[c] = -CUDART_INF_F;
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
#pragma unroll
          for (int c = 0; c < kScoreChunks; ++c)
            part[c] = max3(part[c], __uint_as_float(sr[c][e]), __uint_as_float(sr[c][e + 1]));
        }
        if (BIASED) {
          // Every key of an unmasked tile is at or before the row's position: its bias is slope * (from + e).  The
          // reference of the exponent is taken from the raw maxima of 32 columns and the larger of their two end biases:
          // it lies above the true maximum by at most 31 slopes, under 2^100 of range (see `steep`), which costs nothing
          // in fp32 or bf16 and saves the biased scores a pass of their own.
#pragma unroll
          for (int c = 0; c < kScoreChunks; ++c) {
            const float first = fast_slope * (from + (float)(c * 32));
            part[c] = fmaf(part[c], mult, fmaxf(first, first + 31.f * fast_slope));
          }
        }
        mx = fmaxf(part[0], part[1]);
        if (kScoreChunks == 4) mx = fmaxf(mx, fmaxf(part[2], part[3]));
        if (!BIASED) mx *= mult;                                                    // mult > 0
      }
      // The exponent reference only moves when the maximum grew by more than 2^8: P stays within
      // bf16/fp32 range and O needs rescaling (and the wait for the previous P.V) only then.
      float alpha = 1.f;
      if (mx > m + 8.f || m == -CUDART_INF_F) {
        if (mx > m) {
          alpha = fast_exp2(m - mx);                               // 0 on the first finite maximum
          m = mx;
        }
      }
      const float mu = m == -CUDART_INF_F ? 0.f : m;
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
        alive = __all_sync(0xffffffffu, bar_wait(pv_bar(t, j - 1), pv_phase(j - 1), &sh->abort));
        if (!alive) break;
        tc_fence_after();
#pragma unroll 1
        for (int cb = 0; cb < D / 32; ++cb) {
          uint32_t r[32];
          tmem_ld32(o_addr + cb * 32, r);
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
          tmem_st32(o_addr + cb * 32, r);
        }
      }
      // ---- probabilities, 32 columns at a time.  P (bf16, the reference's rounding point before the
      // second product) overwrites the LOWER half of S; every column of S is in registers by now.
      float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      const float2 mult2 = make_float2(mult, mult), neg_mu2 = make_float2(-mu, -mu);
#pragma unroll
      for (int c = 0; c < kScoreChunks; ++c) {
        uint32_t packed[16];
        // the biases of two neighbouring keys, stepped by additions within 32 columns (at most 16 roundings)
        float2 addend = neg_mu2;
        const float2 bias_step = make_float2(2.f * fast_slope, 2.f * fast_slope);
        if (BIASED) {
          const float first = fast_slope * (from + (float)(c * 32)) - mu;
          addend = make_float2(first, first + fast_slope);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 x = __ffma2_rn(make_float2(__uint_as_float(sr[c][2 * i]), __uint_as_float(sr[c][2 * i + 1])), mult2, addend);
          if (BIASED) addend = __fadd2_rn(addend, bias_step);
          const float2 pr2 = make_float2(fast_exp2(x.x), fast_exp2(x.y));
          sum2[i & 1] = __fadd2_rn(sum2[i & 1], pr2);
          packed[i] = pack_bf16(pr2.x, pr2.y);
        }
        tmem_st16_nowait(p_addr + c * 16, packed);
      }
      l = l * alpha + ((sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y));
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();                                      // every lane's P is in tensor memory: one arrival per warp
      if (lane == 0) bar_arrive(&sh->p_full[buf]);
    }
    // The row a thread owns leaves through shared memory, so that a warp stores whole rows: one thread storing its own
    // row 16 bytes at a time touched 32 rows per instruction and took 3 us per CTA.  16-byte chunks are exchanged by row
    // (^ row & 7), which keeps both sides free of bank conflicts.
    if (SHARED) {
      // wait for the products of both tiles (chains): nothing reads the K and V stages any more, they take the O rows
      if (alive && my_tiles > 0) alive = __all_sync(0xffffffffu, bar_wait(pv_bar(t, my_tiles - 1), pv_phase(my_tiles - 1), &sh->abort));
      const bool have = alive && my_tiles > 0;
      tc_fence_after();
      asm volatile("bar.sync 2, %0;\n" ::"n"(kSoftmaxThreads) : "memory");
      constexpr int kRowChunks = D / 4;
      float4* rows = reinterpret_cast<float4*>(s_k);
      float2* states = reinterpret_cast<float2*>(s_k + kTiles * kRows * D * 4);
      int* entries = reinterpret_cast<int*>(states + 2 * kRows);
      static_assert(kTiles * kRows * D * 4 + 2 * kRows * 12 <= (kKRing + kVStages) * kKvTileBytes, "room for the rows");
      states[t * kRows + pr] = make_float2(m, have ? l : 0.f);
      entries[t * kRows + pr] = pr < mv ? listed.z + w0.z * listed.w + head * G + pr % G : -1;
      if (t < kTiles) {
#pragma unroll 1
        for (int cb = 0; cb < D / 32; ++cb) {
          uint32_t r[32];
          if (have) {
            tmem_ld32(o_addr + cb * 32, r);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) r[e] = 0;
          }
#pragma unroll
          for (int c = 0; c < 8; ++c)
            rows[(t * kRows + pr) * kRowChunks + ((cb * 8 + c) ^ (pr & 7))] =
                make_float4(__uint_as_float(r[c * 4]), __uint_as_float(r[c * 4 + 1]), __uint_as_float(r[c * 4 + 2]),
                            __uint_as_float(r[c * 4 + 3]));
        }
      }
      asm volatile("bar.sync 2, %0;\n" ::"n"(kSoftmaxThreads) : "memory");
      // narrow: eight warps over the rows of the one tile, both chains merged; wide: four warps over the rows of each
      for (int row = NARROW ? warp : warp & 3; row < mv; row += NARROW ? 8 : 4) {
        const int at = NARROW ? row : t * kRows + row;
        float2 state = states[at];
        float w_a = 1.f, w_b = 0.f;
        if (NARROW) {
          const float2 other = states[kRows + row];
          float top = state.y > 0.f ? state.x : -CUDART_INF_F;
          if (other.y > 0.f) top = fmaxf(top, other.x);
          w_a = state.y > 0.f ? fast_exp2(state.x - top) : 0.f;
          w_b = other.y > 0.f ? fast_exp2(other.x - top) : 0.f;
          state = make_float2(top, w_a * state.y + w_b * other.y);
        }
        const int64_t entry = entries[at];
        if (lane == 0) *reinterpret_cast<float2*>(p.part_ml + entry * 2) = state;
        for (int c = lane; c < kRowChunks; c += 32) {
          float4 o = rows[at * kRowChunks + (c ^ (row & 7))];
          if (NARROW) {
            const float4 x = rows[(kRows + row) * kRowChunks + (c ^ (row & 7))];
            o = make_float4(w_a * o.x + w_b * x.x, w_a * o.y + w_b * x.y, w_a * o.z + w_b * x.z, w_a * o.w + w_b * x.w);
          }
          *reinterpret_cast<float4*>(p.part_o + entry * D + c * 4) = o;
        }
      }
    } else if (my_tiles > 0) {
      // epilogue: O / l -> bf16 rows of the output, through this tile's own query rows (its last Q.K^T has run)
      if (alive) alive = __all_sync(0xffffffffu, bar_wait(pv_bar(t, my_tiles - 1), pv_phase(my_tiles - 1), &sh->abort));
      uint4* rows = reinterpret_cast<uint4*>(s_q + t * kQTileBytes);
      if (alive) {
        tc_fence_after();
        const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll 1
        for (int cb = 0; cb < D / 32; ++cb) {
          uint32_t r[32];
          tmem_ld32(o_addr + cb * 32, r);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint4 v;
            v.x = pack_bf16(__uint_as_float(r[c * 8 + 0]) * inv, __uint_as_float(r[c * 8 + 1]) * inv);
            v.y = pack_bf16(__uint_as_float(r[c * 8 + 2]) * inv, __uint_as_float(r[c * 8 + 3]) * inv);
            v.z = pack_bf16(__uint_as_float(r[c * 8 + 4]) * inv, __uint_as_float(r[c * 8 + 5]) * inv);
            v.w = pack_bf16(__uint_as_float(r[c * 8 + 6]) * inv, __uint_as_float(r[c * 8 + 7]) * inv);
            rows[pr * kChunks + ((cb * 4 + c) ^ (pr & 7))] = v;
          }
        }
      }
      asm volatile("bar.sync %0, 128;\n" ::"r"(2 + t) : "memory");         // the four warps of this tile
      if (alive) {
        constexpr int kRowsAtOnce = 32 / kChunks;
        const int c = lane & (kChunks - 1);
        for (int row = (warp & 3) * kRowsAtOnce + lane / kChunks; row < mv; row += 4 * kRowsAtOnce) {
          const uint4 v = rows[row * kChunks + (c ^ (row & 7))];
          const int64_t at = (int64_t)(first_row + t * tile_rows + row / G) * p.out_stride + (int64_t)(head * G + row % G) * D + c * 8;
          for (int dst = 0; dst < p.n_out; ++dst) *reinterpret_cast<uint4*>(p.out[dst] + at) = v;
        }
      }
    }
  } else if (warp < 12) {
    // ================================ K/V loaders =========================================
    const bool is_v = warp >= 10;
    const int lwarp = (warp - 8) & 1;
    const int stages = is_v ? kVStages : kKRing;
    const __nv_bfloat16* base = (is_v ? p.pool_v : p.pool_k) + (int64_t)head * p.slots * D;
    const int32_t* trow = p.table + (int64_t)(p.table_rows ? __ldg(p.table_rows + table_row) : table_row) * p.table_stride;
    const int page_mask = (1 << p.page_shift) - 1;
    const CUtensorMap* map = is_v ? &map_v : &map_k;
    const int head_row = head * (int)p.slots;
    int st = 0, round = 0;                                   // ring position of tile j: stage j % stages, round j / stages
    for (int j = 0; j < n_tiles; ++j) {
      // each loader warp stages half a tile, 32 rows at a time: lanes resolve one slot each, then the
      // warp copies 512 bytes of consecutive rows per instruction (16 bytes a lane)
      constexpr int kWarpRows = kKv / 2, kHalves = kWarpRows / 32;
      int slot[kHalves];
#pragma unroll
      for (int half = 0; half < kHalves; ++half) {
        const int tok = tile_at(j) + lwarp * kWarpRows + half * 32 + lane;
        slot[half] = -1;
        if (tok < kv_end && (!SHARED || tok >= kv_seen)) {
          slot[half] = __ldg(trow + (int64_t)(tok >> p.page_shift) * p.entry_stride) + (tok & page_mask);
          if ((unsigned)slot[half] >= (unsigned)p.slots) {
            if (p.status) atomicOr(p.status, (int)GK_DEV_BAD_TABLE);
            slot[half] = -1;
          }
        }
      }
      // This warp's rows go by TMA when they are whole, in-range boxes of tma_rows slot-contiguous
      // tokens; the two warps of a tile decide independently (every thread arrives once either way).
      const int tok_first = tile_at(j) + lwarp * kWarpRows;
      bool by_tma = p.tma_rows > 0 && (tok_first & (p.tma_rows - 1)) == 0 && tok_first + kWarpRows <= kv_end;
      by_tma = __all_sync(0xffffffffu, by_tma && slot[0] >= 0 && slot[kHalves - 1] >= 0);
      uint64_t* full = is_v ? &sh->v_full[st] : &sh->k_full[st];
      if (round > 0) {   // stage free: K once both Q.K^T of the tile that used it completed, V once both P.V did
        uint64_t* freed = is_v ? &sh->v_free[st] : &sh->k_free[st];
        if (!__all_sync(0xffffffffu, bar_wait_patient(freed, (round - 1) & 1, &sh->abort))) break;
      }
      const uint32_t dst = smem_u32(is_v ? s_v : s_k) + st * kKvTileBytes;
      if (by_tma) {
        if (lane == 0) bar_arrive_expect_tx(full, kWarpRows * D * 2);
        else bar_arrive(full);
        __syncwarp();
        // the lane that holds the first row of a box issues its panels
#pragma unroll
        for (int half = 0; half < kHalves; ++half) {
          const int row = half * 32 + lane;                       // row within this warp's share
          if ((row & (p.tma_rows - 1)) == 0) {
            const uint32_t at = dst + (lwarp * kWarpRows + row) * 128;
#pragma unroll
            for (int panel = 0; panel < G_::kPanels; ++panel)
              tma_load_box(at + panel * kKvPanelBytes, map, panel * 64, head_row + slot[half], full);
          }
        }
      } else {
#pragma unroll
        for (int half = 0; half < kHalves; ++half) {
#pragma unroll 4
          for (int i = 0; i < kChunks; ++i) {                     // 32 rows x kChunks chunks over 32 lanes
            const int at = i * 32 + lane, rr = at / kChunks, c = at & (kChunks - 1);
            const int s = __shfl_sync(0xffffffffu, slot[half], rr);
            cp_async_16(dst + tile_off(lwarp * kWarpRows + half * 32 + rr, c, kKvPanelBytes),
                        base + (int64_t)(s < 0 ? 0 : s) * D + c * 8, s < 0 ? 0 : 16);
          }
        }
        bar_arrive_on_copies(full);
      }
      if (++st == stages) {
        st = 0;
        ++round;
      }
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
  } else if (warp == 12 && lane == 0) {
    // ================================ MMA issue ===========================================
    const uint32_t q_addr = smem_u32(s_q), k_base = smem_u32(s_k), v_base = smem_u32(s_v);
    const int nt[2] = {nt0, nt1}, begin[2] = {head0, 0};
    bool alive = true;
    // Operand descriptors are built once; a k-step or a ring stage only moves the 14-bit address field (units of
    // 16 bytes) in the lower half, so the issue loop is one 32-bit add per operand and the MMA itself.
    const uint64_t q_desc = umma_desc(q_addr, 16, 1024), k_desc = umma_desc(k_base, 16, 1024);
    const uint64_t v_desc = umma_desc(v_base, kKvPanelBytes, 1024);
    const uint32_t q_lo = (uint32_t)q_desc, k_lo = (uint32_t)k_desc, v_lo = (uint32_t)v_desc;
    const uint32_t qk_hi = (uint32_t)(q_desc >> 32), v_hi = (uint32_t)(v_desc >> 32);      // K's upper half equals Q's
    constexpr uint32_t kStageStep = kKvTileBytes >> 4;
    // S[buf] = Q[t] . K[stage]^T ; O[t] += P[buf] . V[stage]
    auto issue_qk = [&](int t, int buf, int stage) {
      const uint32_t a = q_lo + t * (kQTileBytes >> 4), b = k_lo + stage * kStageStep;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {               // 16 elements of head_dim per step
        const uint32_t a_step = ((k >> 2) * kQPanelBytes + (k & 3) * 32) >> 4;
        const uint32_t b_step = ((k >> 2) * kKvPanelBytes + (k & 3) * 32) >> 4;
        umma_bf16_ss_split(tmem + buf * 128, a + a_step, qk_hi, b + b_step, qk_hi, G_::kIdescQK, k > 0 ? 1u : 0u);
      }
      umma_commit(&sh->s_full[buf]);
    };
    auto issue_pv = [&](int t, int buf, int j, int stage) {
      const uint32_t b = v_lo + stage * kStageStep;
#pragma unroll
      for (int k = 0; k < kKv / 16; ++k) {             // 16 tokens per step: 8 columns of P, 16 rows of V
        umma_bf16_ts_split(tmem + 256 + t * D, tmem + buf * 128 + k * 8, b + k * (2048 >> 4), v_hi, G_::kIdescPV,
                           (j > 0 || k > 0) ? 1u : 0u);
      }
      umma_commit(pv_bar(t, j));
    };
    if (NARROW) {
      // Two chains over alternating KV tiles, Q.K^T two tiles ahead of P.V: QK(0), QK(1), then PV(j), QK(j+2) per tile.
      for (int a = 0; a < 2 && a < n_tiles && alive; ++a) {
        alive = bar_wait(&sh->k_full[a], 0, &sh->abort);
        if (!alive) break;
        fence_async_smem();
        tc_fence_after();
        issue_qk(0, a, a);
        umma_commit(&sh->k_free[a]);
      }
      int ks = 2, kround = 0, vs = 0, vround = 0;
      for (int j = 0; j < n_tiles && alive; ++j) {
        alive = bar_wait(&sh->v_full[vs], vround & 1, &sh->abort) &&
                bar_wait(&sh->p_full[j & 1], (j >> 1) & 1, &sh->abort);
        if (!alive) break;
        fence_async_smem();
        tc_fence_after();
        issue_pv(j & 1, j & 1, j >> 1, vs);
        umma_commit(&sh->v_free[vs]);
        if (j + 2 < n_tiles) {                 // the buffer P.V(j) reads is free once that product has run: in order
          alive = bar_wait(&sh->k_full[ks], kround & 1, &sh->abort);
          if (!alive) break;
          fence_async_smem();
          tc_fence_after();
          issue_qk(0, j & 1, ks);
          umma_commit(&sh->k_free[ks]);
          if (++ks == kKRing) {
            ks = 0;
            ++kround;
          }
        }
        if (++vs == kVStages) {
          vs = 0;
          ++vround;
        }
      }
    } else if (kTiles == 1) {
      // One query tile, two score buffers: Q.K^T runs two KV tiles ahead of P.V, so the tensor pipe has the next
      // tile's scores ready while this tile's softmax runs.  Order: QK(0), QK(1), then PV(j), QK(j+2) per tile.
      for (int a = 0; a < 2 && a < n_tiles && alive; ++a) {
        alive = bar_wait(&sh->k_full[a % kKStages], (a / kKStages) & 1, &sh->abort);
        if (!alive) break;
        fence_async_smem();
        tc_fence_after();
        issue_qk(0, a, a % kKStages);
        umma_commit(&sh->k_free[a % kKStages]);
      }
      int vs = 0, vround = 0;
      for (int j = 0; j < n_tiles && alive; ++j) {
        alive = bar_wait(&sh->v_full[vs], vround & 1, &sh->abort) &&
                bar_wait(&sh->p_full[j & 1], (j >> 1) & 1, &sh->abort);
        if (!alive) break;
        fence_async_smem();
        tc_fence_after();
        issue_pv(0, j & 1, j, vs);
        umma_commit(&sh->v_free[vs]);
        if (j + 2 < n_tiles) {                 // the buffer P.V(j) reads is free once that product has run: in order
          const int ks = (j + 2) % kKStages;
          alive = bar_wait(&sh->k_full[ks], ((j + 2) / kKStages) & 1, &sh->abort);
          if (!alive) break;
          fence_async_smem();
          tc_fence_after();
          issue_qk(0, j & 1, ks);
          umma_commit(&sh->k_free[ks]);
        }
        if (++vs == kVStages) {
          vs = 0;
          ++vround;
        }
      }
    } else {
    if (n_tiles > 0) {
      alive = bar_wait(&sh->k_full[0], 0, &sh->abort);
      if (alive) {
        fence_async_smem();
        tc_fence_after();
        for (int t = 0; t < 2; ++t)
          if (nt[t] > 0 && begin[t] == 0) issue_qk(t, t, 0);
        umma_commit(&sh->k_free[0]);
      }
    }
    int ks = 1 % kKStages, kround = 1 / kKStages, vs = 0, vround = 0;     // ring positions of K tile j+1 and V tile j
    for (int j = 0; j < n_tiles && alive; ++j) {
      const bool more = j + 1 < n_tiles;
      alive = bar_wait(&sh->v_full[vs], vround & 1, &sh->abort);
      if (alive && more) alive = bar_wait(&sh->k_full[ks], kround & 1, &sh->abort);
      if (!alive) break;
      fence_async_smem();
      tc_fence_after();
      for (int t = 0; t < 2 && alive; ++t) {
        const int mine = j - begin[t];                 // this query tile's own count
        if (mine >= 0 && mine < nt[t]) {
          alive = bar_wait(&sh->p_full[t], mine & 1, &sh->abort);
          if (!alive) break;
          tc_fence_after();
          issue_pv(t, t, mine, vs);
        }
        if (mine + 1 >= 0 && mine + 1 < nt[t]) issue_qk(t, t, ks);
      }
      if (!alive) break;
      umma_commit(&sh->v_free[vs]);
      if (more) umma_commit(&sh->k_free[ks]);
      if (++vs == kVStages) {
        vs = 0;
        ++vround;
      }
      if (++ks == kKStages) {
        ks = 0;
        ++kround;
      }
    }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (tid == 0 && sh->abort && p.status) atomicOr(p.status, (int)GK_DEV_WAIT_EXPIRED);
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512));
}

template <int D, bool BIASED, int FORM, bool CAP>
int launch_prefill(PrefillParams& p, int64_t n_work, int page_tokens, cudaStream_t stream) {
  static std::atomic<bool> configured[64];
  const int ready = opt_in_shared_memory(paged_prefill_tc_kernel<D, BIASED, FORM, CAP>, Geo<D>::kSmemBytes, configured);
  if (ready != GK_OK) return ready;
  {
    // Never launch if the register pool of this build cannot satisfy the budgets (the kernel would hang).
    static std::atomic<int> launch_regs{-1};
    int regs = launch_regs.load(std::memory_order_acquire);
    if (regs < 0) {
      cudaFuncAttributes attr;
      if (cudaFuncGetAttributes(&attr, paged_prefill_tc_kernel<D, BIASED, FORM, CAP>) != cudaSuccess) return check_launch();
      regs = attr.numRegs;
      launch_regs.store(regs, std::memory_order_release);
    }
    if (regs * kThreads < kSoftmaxThreads * kSoftmaxRegs + 128 * kLoaderRegs + 128 * kIssueRegs) return GK_ERR_UNSUPPORTED;
  }
  // TMA boxes need slot-contiguous pages of at least 8 tokens and 32-bit row coordinates; a box is at most
  // the rows one loader warp stages.
  alignas(64) CUtensorMap map_k, map_v;
  memset(&map_k, 0, sizeof(map_k));
  memset(&map_v, 0, sizeof(map_v));
  constexpr int kWarpRows = Geo<D>::kKv / 2;
  const int box_rows = page_tokens < kWarpRows ? page_tokens : kWarpRows;
  const int64_t pool_rows = (int64_t)p.kv_heads * p.slots;
  if (page_tokens >= 8 && pool_rows < 0x7fffffffLL && make_pool_map(&map_k, p.pool_k, pool_rows, box_rows, D) &&
      make_pool_map(&map_v, p.pool_v, pool_rows, box_rows, D))
    p.tma_rows = box_rows;
  const int64_t ctas = n_work * p.kv_heads * (Geo<D>::kTiles == 2 ? 1 : 2);
  if (ctas > 0x7fffffffLL) return GK_ERR_UNSUPPORTED;
  if (FORM == kRowsForm)
    paged_prefill_tc_kernel<D, BIASED, FORM, CAP><<<(unsigned)ctas, kThreads, Geo<D>::kSmemBytes, stream>>>(p, map_k, map_v);
  else
    launch_after_predecessor(paged_prefill_tc_kernel<D, BIASED, FORM, CAP>, dim3((unsigned)ctas), dim3(kThreads),
                             Geo<D>::kSmemBytes, stream, p, map_k, map_v);
  return check_launch();
}


// Which rows a launch of the kernel serves beyond its work records: a distance bias and row limits, or the listed rows of
// the shared form with the split state that receives their part.
struct PrefillExtras {
  const float* slopes = nullptr;
  const int32_t* row_limits = nullptr;
  const int32_t* list = nullptr;
  bool narrow = false;
  float* part_ml = nullptr;
  float* part_o = nullptr;
};

template <bool BIASED, int FORM, bool CAP>
int launch_prefill_dim(PrefillParams& p, int head_dim, int64_t n_work, int page_tokens, cudaStream_t stream) {
  if (head_dim == 64) return launch_prefill<64, BIASED, FORM, CAP>(p, n_work, page_tokens, stream);
  if (head_dim == 256) return launch_prefill<256, BIASED, FORM == kNarrowForm ? kWideForm : FORM, CAP>(p, n_work, page_tokens, stream);
  return launch_prefill<128, BIASED, FORM, CAP>(p, n_work, page_tokens, stream);
}

template <bool BIASED, int FORM>
int launch_prefill_cap(PrefillParams& p, int head_dim, int64_t n_work, int page_tokens, cudaStream_t stream) {
  return p.softcap > 0.f ? launch_prefill_dim<BIASED, FORM, true>(p, head_dim, n_work, page_tokens, stream)
                         : launch_prefill_dim<BIASED, FORM, false>(p, head_dim, n_work, page_tokens, stream);
}

int prefill_entry(const void* q, int64_t q_row_stride, const void* pool_k, const void* pool_v, int64_t slots,
                  const int32_t* table, int64_t table_stride, int64_t table_entry_stride, int page_tokens,
                  const int32_t* table_rows, const int32_t* work, int64_t n_work, void* const* outs, int n_outs,
                  int64_t out_row_stride, const PrefillExtras& extras, float scale, float softcap, int window, int q_heads,
                  int kv_heads, int head_dim, int32_t* status, gk_stream_t stream) {
  if (n_work == 0) return GK_OK;
  const bool shared = extras.list != nullptr;
  if (shared ? !extras.part_ml || !extras.part_o : !outs || n_outs <= 0 || n_outs > GK_MAX_OUTPUTS) return GK_ERR_INVALID_ARGUMENT;
  if (((reinterpret_cast<uintptr_t>(extras.list) | reinterpret_cast<uintptr_t>(extras.part_o)) & 15) ||
      (reinterpret_cast<uintptr_t>(extras.part_ml) & 7) ||
      ((reinterpret_cast<uintptr_t>(extras.slopes) | reinterpret_cast<uintptr_t>(extras.row_limits)) & 3))
    return GK_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < n_outs; ++i)
    if (!outs[i] || (reinterpret_cast<uintptr_t>(outs[i]) & 15)) return GK_ERR_INVALID_ARGUMENT;
  if (!q || !pool_k || !pool_v || !table || !work || n_work < 0 || slots <= 0 || table_stride < 0 ||
      table_entry_stride <= 0 || page_tokens <= 0 || (page_tokens & (page_tokens - 1)) || q_heads <= 0 || kv_heads <= 0 ||
      !(scale > 0.f) || !(softcap >= 0.f) || (window != -1 && window <= 0))
    return GK_ERR_INVALID_ARGUMENT;
  if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || q_heads % kv_heads != 0 || q_heads / kv_heads > GK_PREFILL_TILE_ROWS ||
      n_work * kv_heads > 0x7fffffffLL)
    return GK_ERR_UNSUPPORTED;
  if (((reinterpret_cast<uintptr_t>(pool_k) | reinterpret_cast<uintptr_t>(pool_v) | reinterpret_cast<uintptr_t>(work)) & 15) ||
      (out_row_stride & 7) || (reinterpret_cast<uintptr_t>(q) & 1))
    return GK_ERR_INVALID_ARGUMENT;
  PrefillParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.pool_k = static_cast<const __nv_bfloat16*>(pool_k);
  p.pool_v = static_cast<const __nv_bfloat16*>(pool_v);
  p.table = table;
  p.table_rows = table_rows;
  p.work = work;
  for (int i = 0; i < n_outs; ++i) p.out[i] = static_cast<__nv_bfloat16*>(outs[i]);
  p.n_out = n_outs;
  p.status = status;
  p.q_stride = q_row_stride;
  p.out_stride = out_row_stride;
  p.slots = slots;
  p.table_stride = table_stride;
  p.entry_stride = table_entry_stride;
  p.scale = scale;
  p.softcap = softcap;
  p.window = window;
  p.page_shift = __builtin_ctz((unsigned)page_tokens);
  p.q_heads = q_heads;
  p.kv_heads = kv_heads;
  p.group = q_heads / kv_heads;
  p.slopes = extras.slopes;
  p.row_limits = extras.row_limits;
  p.list = reinterpret_cast<const int4*>(extras.list);
  p.part_ml = extras.part_ml;
  p.part_o = extras.part_o;
  cudaStream_t at = reinterpret_cast<cudaStream_t>(stream);
  if (shared && extras.narrow)
    return p.slopes ? launch_prefill_cap<true, kNarrowForm>(p, head_dim, n_work, page_tokens, at)
                    : launch_prefill_cap<false, kNarrowForm>(p, head_dim, n_work, page_tokens, at);
  if (shared)
    return p.slopes ? launch_prefill_cap<true, kWideForm>(p, head_dim, n_work, page_tokens, at)
                    : launch_prefill_cap<false, kWideForm>(p, head_dim, n_work, page_tokens, at);
  return p.slopes || p.row_limits ? launch_prefill_cap<true, kRowsForm>(p, head_dim, n_work, page_tokens, at)
                                  : launch_prefill_dim<false, kRowsForm, false>(p, head_dim, n_work, page_tokens, at);
}

}  // namespace
}  // namespace gk

extern "C" int gk_paged_prefill_tc_multi_bf16(const void* q, int64_t q_row_stride, const void* pool_k,
                                              const void* pool_v, int64_t slots, const int32_t* table,
                                              int64_t table_stride, int64_t table_entry_stride, int page_tokens,
                                              const int32_t* table_rows, const int32_t* work, int64_t n_work,
                                              void* const* outs, int n_outs, int64_t out_row_stride, float scale,
                                              float softcap, int window, int q_heads, int kv_heads, int head_dim,
                                              int32_t* status, gk_stream_t stream) {
  return gk::prefill_entry(q, q_row_stride, pool_k, pool_v, slots, table, table_stride, table_entry_stride, page_tokens,
                           table_rows, work, n_work, outs, n_outs, out_row_stride, gk::PrefillExtras{}, scale, softcap,
                           window, q_heads, kv_heads, head_dim, status, stream);
}

extern "C" int gk_paged_prefill_tc_biased_multi_bf16(const void* q, int64_t q_row_stride, const void* pool_k,
                                                     const void* pool_v, int64_t slots, const int32_t* table,
                                                     int64_t table_stride, int64_t table_entry_stride, int page_tokens,
                                                     const int32_t* table_rows, const int32_t* work, int64_t n_work,
                                                     void* const* outs, int n_outs, int64_t out_row_stride,
                                                     const float* slopes, const int32_t* row_limits, float scale,
                                                     float softcap, int window, int q_heads, int kv_heads, int head_dim,
                                                     int32_t* status, gk_stream_t stream) {
  gk::PrefillExtras extras;
  extras.slopes = slopes;
  extras.row_limits = row_limits;
  return gk::prefill_entry(q, q_row_stride, pool_k, pool_v, slots, table, table_stride, table_entry_stride, page_tokens,
                           table_rows, work, n_work, outs, n_outs, out_row_stride, extras, scale, softcap, window, q_heads,
                           kv_heads, head_dim, status, stream);
}

extern "C" int gk_shared_prefix_attn_bf16(const void* q, int64_t q_row_stride, const void* pool_k, const void* pool_v,
                                          int64_t slots, const int32_t* table, int64_t table_stride,
                                          int64_t table_entry_stride, int page_tokens, const int32_t* table_rows,
                                          const int32_t* prefix_work, int64_t n_prefix_work, int form,
                                          const int32_t* prefix_rows, float* part_ml, float* part_o, const float* slopes,
                                          float scale, float softcap, int window, int q_heads, int kv_heads, int head_dim, int32_t* status,
                                          gk_stream_t stream) {
  if (n_prefix_work == 0) return GK_OK;
  if (!prefix_rows || q_heads <= 0 || kv_heads <= 0 || q_heads / kv_heads > GK_MAX_PACKED_ROWS)
    return prefix_rows && q_heads > 0 && kv_heads > 0 ? GK_ERR_UNSUPPORTED : GK_ERR_INVALID_ARGUMENT;
  gk::PrefillExtras extras;
  extras.slopes = slopes;
  extras.list = prefix_rows;
  extras.narrow = (form & GK_SHARED_ONE_TILE) != 0;
  extras.part_ml = part_ml;
  extras.part_o = part_o;
  return gk::prefill_entry(q, q_row_stride, pool_k, pool_v, slots, table, table_stride, table_entry_stride, page_tokens,
                           table_rows, prefix_work, n_prefix_work, nullptr, 0, 8, extras, scale, softcap, window, q_heads,
                           kv_heads, head_dim, status, stream);
}

extern "C" int gk_paged_prefill_tc_bf16(const void* q, int64_t q_row_stride, const void* pool_k, const void* pool_v,
                                        int64_t slots, const int32_t* table, int64_t table_stride,
                                        int64_t table_entry_stride, int page_tokens, const int32_t* table_rows,
                                        const int32_t* work, int64_t n_work, void* out, int64_t out_row_stride,
                                        float scale, float softcap, int window, int q_heads, int kv_heads, int head_dim,
                                        int32_t* status, gk_stream_t stream) {
  void* const outs[1] = {out};
  return gk_paged_prefill_tc_multi_bf16(q, q_row_stride, pool_k, pool_v, slots, table, table_stride, table_entry_stride,
                                        page_tokens, table_rows, work, n_work, outs, 1, out_row_stride, scale, softcap,
                                        window, q_heads, kv_heads, head_dim, status, stream);
}
