// Causal attention of each sequence's new tokens over its pages, the new tokens' own keys and values among them.
//   o[t, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(<q[t, h], k_j> / sqrt(D)),  j <= pos[b] + (number of t in its sequence)
// and, with a gate, o * sigmoid(gate[t, h]).
//
// Two CTAs of a cluster work on one block of queries after another: the G query heads of a key/value head are stacked into the 128 rows of a
// CTA's half of an M = 256 tile (row = token * G + head, 128 / G tokens, what is left of the rows idle).  Per 128 keys, cta_group::2:
//     S[256 x 128]  = Q[256 x D] . K^T           tcgen05.mma, both operands K-major in shared memory, D in TMEM
//     P = exp2(S * scale * log2e - m)             a thread per row, TMEM -> TMEM; bf16, as V is (both operands of a product have one type):
//                                                 2^-8 of itself at most; its sum is fp32
//     O[256 x D]   += P[256 x 128] . V[128 x D]   tcgen05.mma, P from TMEM, V as an MN-major operand, O stays in TMEM
// Each CTA holds 64 keys of a K tile and D/2 columns of a V tile, so a pair fetches a page once.
//
// Pages go straight from the pools into operand layout.  A K-major operand wants its groups of 8 rows at one distance, so K comes in
// half pages: a box {64 columns, 8 slots, D/64 blocks} lands as one group of every column block.  Of V a step of 16 keys is a page: a box
// {64, 16, D/128}.  The page in which a block's keys end is read from a slot below zero, so that its last 16 places hold the last keys and
// what lies in front is filled with zeros: slots behind the end, which may hold anything, are never read (zeros of P do not help against
// NaN in V).  Pages that are none, and those behind the end, are boxes outside the pool, zeros too.  (An infinity or NaN among the values of a
// block's own tokens does make the rows in front of it NaN, whose P is zero there.)
//
// Work is cut by keys: all (sequence, kv head, block of queries) rows stand in a line, each as long as its keys and CA_GAP for what a row costs
// once, and every pair takes an equal stretch.  Lengths are read on the device: nothing the host knows changes from call to call.  A row that a
// cut falls into leaves partial sums (fp32 O, maximum, sum) in the workspace, one per pair, which a second kernel joins in the order of the
// keys; all others are finished here.  No atomics, so equal calls give equal bits.
//
// Roles of the 16 warps: 0-3, 4-7 exponentials of even and odd tiles; 8-11 O through the gate to the output (or the workspace); 12, 15 issue S
// and PV (even CTA); 13 loads K; 14 walks the line and loads Q and V.  O is rescaled only when a row maximum grows by more than 2^8 (the
// reference may lag; p then stays below 2^8, which changes no relative rounding).
//
// Bound by waits of one role for the other at a tile's hand-overs: at 2 x 2048 tokens the tensor pipe works half of the time, the exponential units a
// quarter; in runs of seconds by the power cap as well.  8 x 2048 tokens over 2048, 8 + 2 heads of 256, 368 to 380 us, 1.09 to 1.12 PFLOP/s of a
// cuBLAS product's 1.67 (440 in seconds-long runs); 2048 over 30 000 416 to 427, 1.22 to 1.25: the ends of a block's row cost what three tiles do.
// 16 + 4 heads of 128 371.  Small calls are bound by what lies around: 9 us to the first product, some 4 for the second kernel; 1 x 64 tokens over
// 500 17 us.
// (128 keys a tile: two S beside an O of 256 columns fill tensor memory.  Pairs: half the bytes per CTA of K and V through the L2.)
// Every wait is bounded; on expiry the device error flag is set and the CTA drains.
#include "chunk.cuh"

namespace b200 {

constexpr int CA_TKV = 128;                          // keys of a tile
constexpr int CA_THREADS = 512;
constexpr int CA_SOFTMAX_WARPS = 8, CA_OUT_WARPS = 4;
constexpr int CA_ITEMS = 4;                          // pieces in flight per pair
constexpr int CA_REGS_SOFTMAX = 160, CA_REGS_OUT = 120, CA_REGS_ISSUE = 64;
constexpr int CA_REGS = 65536 / CA_THREADS;          // what __launch_bounds__ leaves a thread, and ptxas gives (the host checks)
static_assert(2 * CA_REGS_SOFTMAX + CA_REGS_OUT + CA_REGS_ISSUE <= CA_THREADS / 128 * CA_REGS, "shares of the registers the CTA is launched with");
constexpr uint32_t CA_TMEM_COLS = 512;               // two or three S of 128 (P over their first 64), O in the last D
constexpr float CA_TAU = 8.0f;                       // lazy-rescale threshold (log2 domain)
// How the line is cut; us with this value and with others.
constexpr int CA_GAP = 384;                          // what a row costs once, in keys: 2 x 1000 tokens over 500 to 5000 75, 192: 77, 768: 78
constexpr int CA_MIN_SHARE = 192;                    // least stretch for a pair: 1 x 128 over 300 16.6, 320: 22.5
constexpr int CA_WHOLE = 1792;                       // rows up to this long are not cut, to join one costs as much as the pairs may differ: 16 x 256
                                                     // over 1000 62, 900: 75; 32 x 60 over 700 32, 900: 43
constexpr int CA_WHOLE_FEW = 640;                    // the same where rows are fewer than pairs: 1 x 64 over 1200 18.7, 1792: 33; 4 x 200 over 0 16, 320: 18
constexpr int CA_STAGE = 3, CA_STAGE_BYTES = 32 * 64;  // buffers of an output warp: 32 columns of its 32 rows, first the gates, then the output

template <int DIM>
struct ChunkShape {
  static constexpr int BLOCKS = DIM / 64;
  static constexpr int Q_BYTES = 128 * DIM * 2;
  static constexpr int KV_BYTES = CA_TKV / 2 * DIM * 2;  // half a tile: K 64 keys, V DIM/2 columns
  // Buffers of S and P, what O leaves of tensor memory, and as many stages of K and of V: that S of a tile is done says that its K is free too,
  // that PV is, its V.  (Signals of their own for four stages of 128 dimensions: 8 x 2048 tokens over 2048 418 us, so 396.)
  static constexpr int BUFFERS = DIM == 256 ? 2 : 3;
  static constexpr int SMEM = Q_BYTES + 2 * BUFFERS * KV_BYTES + CA_OUT_WARPS * CA_STAGE * CA_STAGE_BYTES;
};

// ----------------------------------------------------------------------------- a pair's pieces, read by every role of a CTA
struct ChunkItem {
  int tile0, tiles;    // key tiles of the piece (tiles 0: no more)
  int row0, count;     // packed row of the block's first token, its tokens
  int b, h;
  int key0, keys;      // keys that its first and its last token see
  int slot;            // place of the partial sums, -1: the piece is the whole row
};

template <int DIM, bool GATED>
__global__ void __launch_bounds__(CA_THREADS, 1)
chunk_pair_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const __grid_constant__ ChunkParams p) {
  using Shape = ChunkShape<DIM>;
  constexpr int NB = Shape::BUFFERS, KV_BYTES = Shape::KV_BYTES, BLOCKS = Shape::BLOCKS;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // `lead_*`: waited for by the issuers, in the even CTA of the pair; the others are each CTA's own
  __shared__ uint64_t lead_k[NB], lead_v[NB], lead_q, free_q, lead_p[NB][2], lead_o, lead_s[NB], bar_s[NB], bar_pv[NB],
      bar_m[4][2][2], bar_l[CA_ITEMS], item_full[CA_ITEMS], item_free[CA_ITEMS];
  __shared__ uint32_t tmem_slot;
  __shared__ ChunkItem items[CA_ITEMS];
  __shared__ float row_ref[2][2][128];                // [tile parity][item parity][row]: the reference of the last tile of that parity
  __shared__ float row_end[CA_ITEMS][2][2][128];      // [item][tile parity][reference, sum][row]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = static_cast<int>(cluster_ctarank()), per_cta = p.per / 2;  // query tokens of this CTA
  uint8_t* q_s = smem_raw;
  uint8_t* k_s = q_s + Shape::Q_BYTES;
  uint8_t* v_s = k_s + NB * KV_BYTES;
  uint8_t* out_s = v_s + NB * KV_BYTES;
  bool ok = (smem_u32(smem_raw) & 1023u) == 0;        // swizzled tiles need it; always so with __align__(1024)

  pdl_trigger();                                      // the kernel that joins partial sums waits for this grid before it reads anything
  if (tid == 0) {
    mbar_init(&lead_q, 1);
    mbar_init(&free_q, 1);
    mbar_init(&lead_o, 2 * CA_OUT_WARPS);
    for (int i = 0; i < NB; ++i) {
      mbar_init(&lead_k[i], 1);
      mbar_init(&lead_v[i], 1);
      mbar_init(&lead_p[i][0], CA_SOFTMAX_WARPS);     // the warps of one parity in both CTAs
      mbar_init(&lead_p[i][1], CA_SOFTMAX_WARPS);
      mbar_init(&lead_s[i], 1);
      mbar_init(&bar_s[i], 1);
      mbar_init(&bar_pv[i], 1);
    }
    for (int i = 0; i < 4; ++i)
      for (int n = 0; n < 4; ++n) mbar_init(&bar_m[i][n >> 1][n & 1], 1);
    for (int i = 0; i < CA_ITEMS; ++i) {
      mbar_init(&bar_l[i], CA_SOFTMAX_WARPS);
      mbar_init(&item_full[i], 1);
      mbar_init(&item_free[i], CA_SOFTMAX_WARPS + CA_OUT_WARPS + 1 + (rank == 0 ? 2 : 0));
    }
    mbar_fence_init();
  }

  // ---- the walk along this pair's stretch (warp 14); both CTAs of a pair find the same pieces
  const int pairs = gridDim.x >> 1, me = blockIdx.x >> 1;
  ChunkRow row = {};
  int64_t from = 0, to = 0;
  auto piece = [&](ChunkItem& it) {                   // the next piece with any tiles
    it.tiles = 0;
    while (row.b < p.batch && row.at < to) {
      const int keys = row.keys(p), all = (keys + CA_TKV - 1) / CA_TKV;
      const int t0 = row.cut<CA_TKV>(p, from, all), t1 = row.cut<CA_TKV>(p, to, all);
      const int first = row.j * p.per;
      it.tile0 = t0, it.tiles = t1 - t0;
      it.row0 = row.q.start + first, it.count = min(p.per, row.q.n - first);
      it.b = row.b, it.h = row.h;
      it.key0 = row.q.s + first + 1, it.keys = keys;
      it.slot = it.tiles == all ? -1 : 2 * me + (row.at < from ? 0 : 1);
      chunk_next(p, row);
      if (it.tiles > 0) return;
    }
  };
  if (warp == 12) tmem_alloc_pair(&tmem_slot, CA_TMEM_COLS);
  if (warp == 13 && lane == 0) {
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  tc_fence_before_sync();
  cluster_arrive();                                   // barriers of both CTAs are set up, tensor memory is there
  ChunkItem it0;
  if (warp == 14) {                                   // while the pair meets
    const int per_lane = (p.batch + 31) / 32;
    int64_t in_front, mine;
    const int64_t line = chunk_line(p, lane, per_lane, in_front, mine), share = chunk_share(p, line, pairs);
    from = min(line, me * share);
    to = min(line, from + share);
    row.b = p.batch;
    if (from < line) row = chunk_find(p, from, lane, per_lane, in_front, mine);
    piece(it0);
  }
  cluster_wait();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  const uint32_t tmem_o = tmem + NB * CA_TKV;

  // item i of this pair; the whole warp
  auto release = [&](int i) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_free[i & (CA_ITEMS - 1)]);
  };
  auto fetch = [&](int i, ChunkItem& it, bool keep = false) {
    ok = warp_wait_bounded(&item_full[i & (CA_ITEMS - 1)], (i / CA_ITEMS) & 1, ok);
    it.tiles = 0;
    if (ok) it = items[i & (CA_ITEMS - 1)];
    if (!keep) release(i);
    return ok && it.tiles > 0;
  };
  // Pages of a piece, 32 at a time (four tiles), one per lane; the next window is asked for early.  -1: none, or behind the end.
  auto page_window = [&](const ChunkItem& it, int window) {
    const int lp = window * 32 + lane;
    int id = -1;
    if (lp <= (it.keys - 1) / PAGE && lp < p.max_pages) id = p.block_table[it.b * p.bt_b + lp];
    return id >= 0 && id < p.num_pages ? id : -1;
  };

  if (warp >= 12) {
    set_registers<CA_REGS_ISSUE, CA_REGS>();
    ChunkItem it;
    if (warp == 14) {
      // ---------------------------------------------------------------- the pieces; TMA producer: Q, and this CTA's columns of every V tile
      auto make = [&](int i, ChunkItem& it) {
        if (i > 0) piece(it);
        if (i >= CA_ITEMS) ok = warp_wait_bounded(&item_free[i & (CA_ITEMS - 1)], (i / CA_ITEMS - 1) & 1, ok);
        if (ok && lane == 0) {
          items[i & (CA_ITEMS - 1)] = it;
          mbar_arrive(&item_full[i & (CA_ITEMS - 1)]);
        }
        return ok && it.tiles > 0;
      };
      const uint32_t full_q = peer_smem(&lead_q, 0), full_v = peer_smem(&lead_v[0], 0);
      const uint32_t q_rows = per_cta * p.group;
      ChunkItem next;
      it = it0;
      bool more = make(0, it);
      int i = 0, g = 0;
      for (; more; ++i, it = next) {
        int ids = page_window(it, it.tile0 >> 2), later = -1;
        if (i > 0) ok = warp_wait_bounded(&free_q, (i - 1) & 1, ok);  // the last S of the item in front has read Q
        if (!ok) break;
        if (lane == 0) {
          if (rank == 0) mbar_expect_tx(&lead_q, 2 * BLOCKS * q_rows * 128);
#pragma unroll 1
          for (int c = 0; c < BLOCKS; ++c)
            tma_load_5d_pair(q_s + c * 16384, &map_q, 0, 0, it.h, it.row0 + rank * per_cta, c, full_q);
        }
        more = false;
        const int last_page = (it.keys - 1) / PAGE, below = it.keys - PAGE * (last_page + 1);  // slot at which the last page is read
        for (int j = 0; j < it.tiles; ++j, ++g) {
          const int tile = it.tile0 + j, st = g % NB;
          if (j == 0 || (tile & 3) == 0) {
            if (j > 0) ids = later;
            later = page_window(it, (tile >> 2) + 1);
          }
          if (g >= NB) ok = warp_wait_bounded(&bar_pv[st], (g / NB - 1) & 1, ok);  // PV of tile g - NB done: its V is free
          if (!ok) break;
          if (rank == 0 && lane == 0) mbar_expect_tx(&lead_v[st], 2 * KV_BYTES);
          const int id = __shfl_sync(0xffffffffu, ids, (tile & 3) * 8 + (lane & 7));
          if (lane < 8)
            tma_load_5d_pair(v_s + st * KV_BYTES + lane * (KV_BYTES / 8), &map_v, 0, tile * 8 + lane == last_page ? below : 0,
                             rank * (BLOCKS / 2), it.h, id, full_v + st * 8);
          __syncwarp();
          if (j == 0) {
            more = make(i + 1, next);
            if (more && lane < BLOCKS) tma_prefetch_5d(&map_q, 0, 0, next.h, next.row0 + rank * per_cta, lane);
          }
        }
        if (!ok) break;
      }
      // the products' last signals have arrived before this CTA may leave
      for (int t = max(0, g - NB); t < g; ++t) ok = warp_wait_bounded(&bar_pv[t % NB], (t / NB) & 1, ok);
      if (i > 0) ok = warp_wait_bounded(&free_q, (i - 1) & 1, ok);
    } else if (warp == 13) {
      // ---------------------------------------------------------------- TMA producer: this CTA's 64 keys of every K tile
      const uint32_t full_k = peer_smem(&lead_k[0], 0);
      int g = 0;
      for (int i = 0; fetch(i, it); ++i) {
        int ids = page_window(it, it.tile0 >> 2), later = -1;
        const int last_page = (it.keys - 1) / PAGE, below = it.keys - PAGE * (last_page + 1);
        for (int j = 0; j < it.tiles; ++j, ++g) {
          const int tile = it.tile0 + j, st = g % NB;
          if (j == 0 || (tile & 3) == 0) {
            if (j > 0) ids = later;
            later = page_window(it, (tile >> 2) + 1);
          }
          if (g >= NB) ok = warp_wait_bounded(&bar_s[st], (g / NB - 1) & 1, ok);  // S of tile g - NB done: its K is free
          if (!ok) break;
          if (rank == 0 && lane == 0) mbar_expect_tx(&lead_k[st], 2 * KV_BYTES);
          const int nth = rank * 4 + ((lane >> 1) & 3);                 // page of the tile; a lane loads half of it
          const int id = __shfl_sync(0xffffffffu, ids, (tile & 3) * 8 + nth);
          if (lane < 8)
            tma_load_5d_pair(k_s + st * KV_BYTES + lane * (KV_BYTES / 8), &map_k, 0, (tile * 8 + nth == last_page ? below : 0) + (lane & 1) * 8,
                             0, it.h, id, full_k + st * 8);
          __syncwarp();
        }
      }
      for (int t = max(0, g - NB); t < g; ++t) ok = warp_wait_bounded(&bar_s[t % NB], (t / NB) & 1, ok);
    } else if (warp == 12 && rank == 0) {
      // ---------------------------------------------------------------- issuer of S for the pair (the whole warp walks, lane 0 issues)
      const bool leader = lane == 0;
      const uint32_t idesc_s = idesc_bf16_f32(256, CA_TKV, false, false);
      const uint32_t q_addr = smem_u32(q_s), k_addr = smem_u32(k_s);
      for (int i = 0, g = 0; fetch(i, it); ++i) {
        ok = warp_wait_cluster(&lead_q, i & 1, ok);
        for (int j = 0; j < it.tiles; ++j, ++g) {
          const int s = g % NB;
          ok = ok && mbar_wait_bounded(&lead_k[s], (g / NB) & 1);
          // S(g) overwrites the buffer whose first columns hold P(g-NB): the PV product that reads them from tensor
          // memory must have COMPLETED, issue order alone does not protect an operand in tensor memory
          if (g >= NB) ok = ok && mbar_wait_bounded(&bar_pv[s], (g / NB - 1) & 1);
          ok = __all_sync(0xffffffffu, ok) != 0;
          if (!ok) break;
          tc_fence_after_sync();
          // (128 dimensions: issued slowly, so that PV finds a place between two S: 8 x 2048 tokens over 2048 418 us by fours, 491 unrolled, 380 by
          // twos; 256: 463 us by fours for 2048 tokens over 30 000, 440 unrolled)
#pragma unroll(DIM == 256 ? 16 : 2)
          for (int ks = 0; ks < DIM / 16; ++ks)
            umma_ss_pair(tmem + s * CA_TKV, smem_desc_sw128(q_addr + (ks >> 2) * 16384 + (ks & 3) * 32, 16, 1024),
                         smem_desc_sw128(k_addr + s * KV_BYTES + (ks >> 2) * 1024 + (ks & 3) * 32, 16, DIM * 16), idesc_s, ks > 0, leader);
          umma_commit_pair(&bar_s[s], leader);
          if (j + 1 == it.tiles) umma_commit_pair(&free_q, leader);
          if (leader) mbar_arrive(&lead_s[s]);
        }
      }
    } else if (warp == 12) {
      // ---------------------------------------------------------------- what the second kernel needs to know of the row that the stretch ends in
      const int per_lane = (p.batch + 31) / 32;
      int64_t in_front, mine;
      const int64_t line = chunk_line(p, lane, per_lane, in_front, mine), share = chunk_share(p, line, pairs), end = (me + 1) * share;
      ChunkCut cut = {};
      if (end < line) {
        const ChunkRow r = chunk_find(p, end, lane, per_lane, in_front, mine);
        if (r.at < end && r.at >= end - share) {
          const int all = (r.keys(p) + CA_TKV - 1) / CA_TKV, begun = r.j * p.per;
          cut.row0 = r.q.start + begun, cut.count = min(p.per, r.q.n - begun), cut.h = r.h;
          cut.first = me;
          cut.begin = r.first_stretch<CA_TKV>(p, share, all);
          cut.last = r.last_stretch<CA_TKV>(p, share, all);
        }
      }
      if (lane == 0) p.cuts[me] = cut;
    } else if (warp == 15 && rank == 0) {
      // ---------------------------------------------------------------- issuer of PV for the pair
      // Inside an item S of the tile behind goes into the pipe first: PV has its operand later anyway.
      const bool leader = lane == 0;
      const uint32_t idesc_o = idesc_bf16_f32(256, DIM, false, true);
      const uint32_t v_addr = smem_u32(v_s);
      int items_done = 0;
      for (int i = 0, g = 0; fetch(i, it); ++i) {
        for (int j = 0; j < it.tiles; ++j, ++g) {
          const int s = g % NB;
          ok = ok && mbar_wait_bounded(&lead_s[s], (g / NB) & 1);
          if (j + 1 < it.tiles) ok = ok && mbar_wait_bounded(&lead_s[(g + 1) % NB], ((g + 1) / NB) & 1);
          ok = ok && mbar_wait_bounded(&lead_v[s], (g / NB) & 1);
          if (j == 0 && i > 0) ok = ok && mbar_wait_bounded(&lead_o, (i - 1) & 1);  // O of the item in front has been read
          ok = __all_sync(0xffffffffu, ok) != 0;
#pragma unroll
          for (int half = 0; half < 2; ++half) {  // the second 64 keys' exponentials are computed under the first 64's product
            ok = warp_wait_bounded(&lead_p[s][half], (g / NB) & 1, ok);
            if (!ok) break;
            tc_fence_after_sync();
#pragma unroll
            for (int kt = half * 4; kt < half * 4 + 4; ++kt)
              umma_ts_pair(tmem_o, tmem + s * CA_TKV + kt * 8,  // P: 16 keys = 8 packed columns per step
                           smem_desc_sw128(v_addr + s * KV_BYTES + kt * (KV_BYTES / 8), 2048, 1024), idesc_o, j > 0 || kt > 0, leader);
          }
          if (!ok) break;
          umma_commit_pair(&bar_pv[s], leader);
        }
        items_done = i + 1;
      }
      if (items_done > 0) ok = warp_wait_bounded(&lead_o, (items_done - 1) & 1, ok);  // the other CTA's last signal
    }
    if (!ok) {
      if (lane == 0) atomicExch(p.err, 1);
      // copies in flight signal barriers that may be the other CTA's: give them their time before the shared memory goes away
      const uint64_t t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 100000) __nanosleep(1000);
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------------------ output of an item, or its partial sums
    set_registers<CA_REGS_OUT, CA_REGS>();
    const int r = tid - 8 * 32;                // TMEM lane; row = token * group + head
    const uint32_t lane_base = static_cast<uint32_t>(r & ~31) << 16;
    const uint32_t read_o = peer_smem(&lead_o, 0);
    uint8_t* stage = out_s + (warp - 8) * (CA_STAGE * CA_STAGE_BYTES);  // of [32 rows][32 columns] bf16, chunk k of a row at k ^ (row / 2 % 4)
    const int tok = r / p.group;
    // the rows whose 16 bytes this lane stores: 8 to an instruction, 4 lanes each
    int store_tok[4], store_col[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int rr = (r & ~31) + n * 8 + (lane >> 2);
      store_tok[n] = rr / p.group;
      store_col[n] = (rr - store_tok[n] * p.group) * DIM + (lane & 3) * 8;
    }
    ChunkItem it;
    for (int i = 0, g = 0; fetch(i, it, true); ++i) {
      g += it.tiles;
      const int slot = i & (CA_ITEMS - 1);
      const int count = min(per_cta, it.count - rank * per_cta);  // tokens of this CTA
      const bool valid = tok < count, whole = it.slot < 0;
      const int64_t t0 = it.row0 + rank * per_cta;
      const int64_t col0 = static_cast<int64_t>(it.h) * p.group * DIM;
      // the gates of 32 columns, in the places of the output; CA_STAGE pieces on their way
      auto load_gate = [&](int c) {
        if (c < DIM / 32) {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int rr = n * 8 + (lane >> 2);
            if (store_tok[n] < count)
              cp_async16(stage + c % CA_STAGE * CA_STAGE_BYTES + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4),
                         p.gate + (t0 + store_tok[n]) * p.gate_t + col0 + store_col[n] + c * 32);
          }
        }
        cp_async_commit();
      };
      if (GATED && whole) {
#pragma unroll
        for (int c = 0; c < CA_STAGE; ++c) load_gate(c);
      }
      ok = warp_wait_bounded(&bar_l[slot], (i / CA_ITEMS) & 1, ok);
      // bar_l is behind S of the item's last tile, S behind PV that read its buffer before: the phase in front of this one is over
      ok = warp_wait_bounded(&bar_pv[(g - 1) % NB], ((g - 1) / NB) & 1, ok);
      if (!ok) break;
      tc_fence_after_sync();
      // even and odd tiles summed against references of their own; O stands at the larger, the last tile's.  A piece in which a row sees
      // nothing has -inf there, and zeros in O and sum
      const float m0 = row_end[slot][0][0][r], m1 = row_end[slot][1][0][r], m = fmaxf(m0, m1), at = m == -INFINITY ? 0.f : m;
      const float l = row_end[slot][0][1][r] * ex2_fast(m0 - at) + row_end[slot][1][1][r] * ex2_fast(m1 - at);
      const uint64_t inv2 = f32x2(1.f / l, 1.f / l);
      if (!whole && valid) reinterpret_cast<float2*>(p.part_ml)[static_cast<int64_t>(it.slot) * 256 + rank * 128 + r] = make_float2(m, l);
      float4* part = reinterpret_cast<float4*>(p.part_o) + (static_cast<int64_t>(max(it.slot, 0)) * (DIM / 4)) * 256 + rank * 128 + r;
      __nv_bfloat16* out = p.out + t0 * p.out_t + col0;
#pragma unroll 1
      for (int c = 0; c < DIM / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(tmem_o + lane_base + c * 32, o);
        if (GATED && whole) {
          cp_async_wait_but<CA_STAGE - 1>();
          __syncwarp();
        }
        tmem_ld_wait();
        if (c == DIM / 32 - 1) {  // O is read: the next item's first product may overwrite it
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_plain(read_o);
        }
        if (!whole) {
          if (valid) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              part[(c * 8 + k) * 256] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]), __uint_as_float(o[4 * k + 2]),
                                                    __uint_as_float(o[4 * k + 3]));
          }
          continue;
        }
        uint8_t* buf = stage + c % CA_STAGE * CA_STAGE_BYTES;
        uint4* mine = reinterpret_cast<uint4*>(buf + lane * 64);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t w[4];
          uint32_t gw[4] = {};
          if (GATED) {
            const uint4 gs = mine[k ^ ((lane >> 1) & 3)];
            gw[0] = gs.x, gw[1] = gs.y, gw[2] = gs.z, gw[3] = gs.w;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint64_t x = f32x2_mul(f32x2(o[k * 8 + e * 2], o[k * 8 + e * 2 + 1]), inv2);
            if (GATED) x = gate_pair(x, gw[e]);
            w[e] = pack_bf16x2(x);
          }
          mine[k ^ ((lane >> 1) & 3)] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int rr = n * 8 + (lane >> 2);
          const uint4 v = *reinterpret_cast<const uint4*>(buf + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4));
          if (store_tok[n] < count) *reinterpret_cast<uint4*>(out + store_tok[n] * p.out_t + store_col[n] + c * 32) = v;
        }
        __syncwarp();
        if (GATED) load_gate(c + CA_STAGE);
      }
      release(i);  // only now: the item's place in the ring is also that of its sums
    }
    if (!ok && lane == 0) atomicExch(p.err, 1);
  } else {
    // ------------------------------------------------------------------ softmax
    set_registers<CA_REGS_SOFTMAX, CA_REGS>();
    // Warps 0-3 take the even tiles of the pair's stream, warps 4-7 the odd ones, one thread per row: while one of the two warps of a
    // scheduler waits for its scores, its row's reference or the store of P, the other has its exponentials computed.
    const int quarter = warp & 3, par = warp >> 2;
    const int r = 32 * quarter + lane;         // TMEM lane; row = token * group + head
    const uint32_t lane_base = static_cast<uint32_t>(32 * quarter) << 16;
    const uint32_t ready_p0 = peer_smem(&lead_p[0][0], 0);
    const float scale = p.scale_log2;
    const int tok = rank * per_cta + r / p.group;
    uint32_t refs[2] = {0, 0};                 // references taken over from the other warp so far, in even and odd items
    ChunkItem it;
    for (int i = 0, g0 = 0; fetch(i, it); ++i) {
      const int see = min(it.key0 + min(tok, it.count - 1), it.keys);  // keys that this row sees
      const int last_page = (it.keys - 1) / PAGE, shift = PAGE * (last_page + 1) - it.keys;
      float m_ref = -INFINITY, l_run = 0.f;
      for (int j = (g0 ^ par) & 1; j < it.tiles; j += 2) {
        const int g = g0 + j, buf = g % NB, key = (it.tile0 + j) * CA_TKV;
        const uint32_t tmem_s = tmem + lane_base + buf * CA_TKV, ready_p = ready_p0 + buf * 16;
        ok = warp_wait_bounded(&bar_s[buf], (g / NB) & 1, ok);
        if (!ok) break;
        tc_fence_after_sync();
        // columns up to lim; the last page's keys stand at its end, `shift` places further
        const int lim = see - 1 - key, tail = last_page * PAGE - key;
        const bool edge = __any_sync(0xffffffffu, lim < CA_TKV - 1 || tail < CA_TKV);
        // the row maximum of the raw scores; the scale (> 0) is folded into the exponent below
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll 1
        for (int c0 = 0; c0 < CA_TKV; c0 += 64) {
          uint32_t s[2][32];
          tmem_ld32(tmem_s + c0, s[0]);
          tmem_ld32(tmem_s + c0 + 32, s[1]);
          tmem_ld_wait();
          if (edge) {  // back into tensor memory, where the second pass finds it
#pragma unroll
            for (int page = 0; page < 4; ++page) {
              const int at = c0 + page * PAGE, behind = at == tail ? shift : 0;
              const int last = at > tail ? -1 : min(lim + behind - at, PAGE - 1);  // of the 16 columns, those from `behind` to it
              const uint32_t seen = last < 0 ? 0u : ((2u << last) - 1u) & (0xffffu << behind);
#pragma unroll
              for (int c = 0; c < PAGE; ++c)
                if ((seen & (1u << c)) == 0) s[page >> 1][(page & 1) * PAGE + c] = 0xff800000u;  // -inf
            }
            tmem_st32(tmem_s + c0, s[0]);
            tmem_st32(tmem_s + c0 + 32, s[1]);
          }
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            mx0 = fmaxf(mx0, fmaxf(__uint_as_float(s[0][c]), __uint_as_float(s[0][c + 1])));
            mx1 = fmaxf(mx1, fmaxf(__uint_as_float(s[1][c]), __uint_as_float(s[1][c + 1])));
          }
        }
        if (edge) tmem_st_wait();
        const float m_tile = fmaxf(mx0, mx1) * scale;
        float m_use = m_tile;
        if (j > 0) {
          ok = warp_wait_bounded(&bar_m[quarter][par ^ 1][i & 1], ((i & 1) ? refs[1]++ : refs[0]++) & 1, ok);
          if (!ok) break;
          const float m_prev = row_ref[par ^ 1][i & 1][r], m_new = fmaxf(m_prev, m_tile);
          const bool need = m_new - m_prev > CA_TAU;  // (-inf behind -inf: NaN, no)
          m_use = need ? m_new : m_prev;
          if (j + 1 < it.tiles) {
            row_ref[par][i & 1][r] = m_use;
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_m[quarter][par][i & 1]);
          }
          if (__any_sync(0xffffffffu, need)) {
            // O must be at rest before it is rescaled: wait for the PV product of the tile in front
            ok = warp_wait_bounded(&bar_pv[(g - 1) % NB], ((g - 1) / NB) & 1, ok);
            if (!ok) break;
            tc_fence_after_sync();
            const float alpha = need ? ex2_fast(m_prev - m_new) : 1.f;
#pragma unroll 1
            for (int c0 = 0; c0 < DIM; c0 += 32) {
              uint32_t o[32];
              tmem_ld32(tmem_o + lane_base + c0, o);
              tmem_ld_wait();
#pragma unroll
              for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
              tmem_st32(tmem_o + lane_base + c0, o);
            }
          }
        } else if (it.tiles > 1) {
          row_ref[par][i & 1][r] = m_use;
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_m[quarter][par][i & 1]);
        }
        const float neg = m_use == -INFINITY ? 0.f : -m_use;  // a row that has seen nothing yet: every p is 2^-inf
        l_run *= ex2_fast(m_ref + neg);        // this parity's sum so far, against the reference of its last tile
        m_ref = m_use;
        // p = 2^(s*scale - m_ref): fp32 for l, bf16 for the PV product, stored as packed columns of the P tile (keys 2c, 2c+1 in
        // column c) over the columns of S that have been read
        const uint64_t sc2 = f32x2(scale, scale), neg2 = f32x2(neg, neg);
        uint64_t sum0 = 0, sum1 = 0;
#pragma unroll 1
        for (int c0 = 0; c0 < CA_TKV; c0 += 64) {
          uint32_t s[2][32];
          tmem_ld32(tmem_s + c0, s[0]);
          tmem_ld32(tmem_s + c0 + 32, s[1]);
          tmem_ld_wait();
          uint32_t w[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const uint64_t x = f32x2_fma(f32x2(s[c >> 4][(2 * c) & 31], s[c >> 4][(2 * c + 1) & 31]), sc2, neg2);
            const uint64_t e = f32x2(ex2_fast(f32x2_lo(x)), ex2_fast(f32x2_hi(x)));
            if (c & 1) sum1 = f32x2_add(sum1, e);
            else sum0 = f32x2_add(sum0, e);
            w[c] = pack_bf16x2(e);
          }
          tmem_st32(tmem_s + (c0 >> 1), w);
          tmem_st_wait();
          tc_fence_before_sync();              // this warp's TMEM loads/stores before the arrive
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_plain(ready_p + (c0 >> 6) * 8);
        }
        sum0 = f32x2_add(sum0, sum1);
        l_run += f32x2_lo(sum0) + f32x2_hi(sum0);
      }
      if (!ok) break;
      g0 += it.tiles;
      const int slot = i & (CA_ITEMS - 1);
      row_end[slot][par][0][r] = m_ref;
      row_end[slot][par][1][r] = l_run;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_l[slot]);
    }
    if (!ok && lane == 0) atomicExch(p.err, 1);
  }
  tc_fence_before_sync();
  // Nobody reads or signals the other CTA any more: each signal between the two has been waited for.  (A release would wait for the stores
  // of the output too.)
  cluster_started();
  cluster_all_started();
  if (warp == 12) tmem_dealloc_pair(tmem, CA_TMEM_COLS);
}

// Joins the partial sums of the rows that the line's cuts fall into: out = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i, pieces in order.
// Work is handed out in units of 8 rows of a block, and of 32 dimensions where many pieces meet.  How many units there are
// stands in the cuts, which every CTA reads: a grid for all that there could be is mostly CTAs that come and go, a microsecond each.
// Of few pieces a thread takes them all, of a row's 4 dimensions here and there; many are shared among four groups of threads, whose sums meet
// in shared memory.  Bound by the partial sums' way through the L2 and its latency.
constexpr int CJ_THREADS = 256, CJ_ROWS = 8, CJ_GROUPS = 4, CJ_MANY = 12;
constexpr int CJ_GRID = 2;                           // CTAs to an SM (with four, of half the registers, 2 x 1000 tokens 82 us, so 75)
constexpr int CJ_MAX_CUTS = 255;
// A unit of the join: 8 rows of half a block, those of the even CTA first; where many pieces meet, 32 of their dimensions.
template <int DIM>
__device__ __forceinline__ void chunk_join_unit(const ChunkParams& p, const ChunkCut& cut, int unit, int units0, float4* share_o, float2* share_ml) {
  const int tid = threadIdx.x, begin = cut.begin, pieces = cut.last - begin + 1, per_cta = p.per / 2;
  const int parts = pieces < CJ_MANY ? 1 : DIM / 32, part_of = unit % parts;
  unit /= parts;
  const int half = unit >= units0, r0 = (half ? unit - units0 : unit) * CJ_ROWS + (tid & 7);
  const int rows = min(cut.count - half * per_cta, per_cta) * p.group;  // of the half
  auto slot_of = [&](int i) { return static_cast<int64_t>(2 * i + (i == cut.first)); };
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + half * 128 + r0;
  const float4* part = reinterpret_cast<const float4*>(p.part_o) + half * 128 + r0;
  auto load = [&](int piece, int quad) { return __ldcg(part + (slot_of(begin + piece) * (DIM / 4) + quad) * 256); };
  auto place = [&](int64_t& t, int64_t& col) {
    const int tok = r0 / p.group;
    t = cut.row0 + half * per_cta + tok;
    col = static_cast<int64_t>(cut.h * p.group + r0 - tok * p.group) * DIM;
  };
  auto finish = [&](int64_t t, int64_t col, float4 o, float l, uint2 g) {
    const float inv = 1.f / l;
    uint64_t v0 = f32x2(o.x * inv, o.y * inv), v1 = f32x2(o.z * inv, o.w * inv);
    if (p.gate) v0 = gate_pair(v0, g.x), v1 = gate_pair(v1, g.y);
    *reinterpret_cast<uint2*>(p.out + t * p.out_t + col) = make_uint2(pack_bf16x2(v0), pack_bf16x2(v1));
  };
  auto add = [](float4& o, float f, const float4& x) { o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y), o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w); };
  if (pieces < CJ_MANY) {
    if (r0 >= rows) return;
    // a batch of pieces is asked for before any of it is used
    constexpr int MINE = DIM / 128, AT_ONCE = 3;
    float4 o[MINE] = {};
    uint2 g[MINE] = {};
    float m = -INFINITY, l = 0.f;
    int64_t t, col;
    place(t, col);
    if (p.gate) {
#pragma unroll
      for (int k = 0; k < MINE; ++k) g[k] = *reinterpret_cast<const uint2*>(p.gate + t * p.gate_t + col + ((tid >> 3) + k * 32) * 4);
    }
#pragma unroll 1
    for (int i0 = 0; i0 < pieces; i0 += AT_ONCE) {
      float2 x[AT_ONCE];
      float4 y[AT_ONCE][MINE];
      float to = m;
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        x[i] = make_float2(-INFINITY, 0.f);
        if (i0 + i < pieces) {
          x[i] = __ldcg(ml + slot_of(begin + i0 + i) * 256);
#pragma unroll
          for (int k = 0; k < MINE; ++k) y[i][k] = load(i0 + i, (tid >> 3) + k * 32);
        }
      }
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) to = fmaxf(to, x[i].x);
      if (to == -INFINITY) continue;  // the row sees nothing of these pieces
      const float f = ex2_fast(m - to);
      l *= f, m = to;
#pragma unroll
      for (int k = 0; k < MINE; ++k) o[k].x *= f, o[k].y *= f, o[k].z *= f, o[k].w *= f;
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
        if (x[i].x != -INFINITY) {
          const float e = ex2_fast(x[i].x - m);
          l = fmaf(x[i].y, e, l);
#pragma unroll
          for (int k = 0; k < MINE; ++k) add(o[k], e, y[i][k]);
        }
    }
#pragma unroll
    for (int k = 0; k < MINE; ++k) finish(t, col + ((tid >> 3) + k * 32) * 4, o[k], l, g[k]);
    return;
  }
  const int share = tid / (CJ_THREADS / CJ_GROUPS), quad = part_of * 8 + ((tid >> 3) & 7);
  const bool valid = r0 < rows;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto take = [&](float mi, float li, const float4& y) {
    if (mi == -INFINITY) return;  // the row sees nothing of this piece
    const float to = fmaxf(m, mi), f = ex2_fast(m - to), g = ex2_fast(mi - to);
    o.x *= f, o.y *= f, o.z *= f, o.w *= f;
    l = fmaf(l, f, li * g), m = to;
    add(o, g, y);
  };
  if (valid) {
    constexpr int AT_ONCE = 5;
#pragma unroll 1
    for (int i = share; i < pieces; i += CJ_GROUPS * AT_ONCE) {
      float2 x[AT_ONCE];
      float4 y[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int piece = i + k * CJ_GROUPS;
        x[k] = make_float2(-INFINITY, 0.f);
        if (piece < pieces) x[k] = __ldcg(ml + slot_of(begin + piece) * 256), y[k] = load(piece, quad);
      }
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) take(x[k].x, x[k].y, y[k]);
    }
  }
  __syncthreads();
  share_o[tid] = o, share_ml[tid] = make_float2(m, l);
  __syncthreads();
  if (share == 0 && valid) {
#pragma unroll
    for (int k = 1; k < CJ_GROUPS; ++k) {
      const int from = tid + k * (CJ_THREADS / CJ_GROUPS);
      take(share_ml[from].x, share_ml[from].y, share_o[from]);
    }
    int64_t t, col;
    place(t, col);
    finish(t, col + quad * 4, o, l, p.gate ? *reinterpret_cast<const uint2*>(p.gate + t * p.gate_t + col + quad * 4) : make_uint2(0, 0));
  }
}

template <int DIM>
__global__ void __launch_bounds__(CJ_THREADS, CJ_GRID)
chunk_join_kernel(const __grid_constant__ ChunkParams p, int cuts) {
  __shared__ float4 share_o[CJ_THREADS];
  __shared__ float2 share_ml[CJ_THREADS];
  __shared__ ChunkCut all[CJ_MAX_CUTS];
  __shared__ int upto[CJ_THREADS];                    // units of this cut and those before it
  __shared__ int warp_units[CJ_THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, per_cta = p.per / 2;
  auto units_of = [&](const ChunkCut& cut, int half) {
    return (max(min(cut.count - half * per_cta, per_cta), 0) * p.group + CJ_ROWS - 1) / CJ_ROWS;
  };
  pdl_wait();
  int units = 0;
  if (tid < cuts) {
    const ChunkCut cut = p.cuts[tid];
    all[tid] = cut;
    const int pieces = cut.last - cut.begin + 1;
    if (pieces > 1) units = (units_of(cut, 0) + units_of(cut, 1)) * (pieces < CJ_MANY ? 1 : DIM / 32);
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, units, o);
    if (lane >= o) units += up;
  }
  if (lane == 31) warp_units[warp] = units;
  __syncthreads();
  for (int w = 0; w < warp; ++w) units += warp_units[w];
  upto[tid] = units;
  __syncthreads();
  const int total = upto[CJ_THREADS - 1];
  for (int unit = blockIdx.x; unit < total; unit += gridDim.x) {
    int at = 0;                                       // cuts that are done with before this unit
#pragma unroll
    for (int step = CJ_THREADS / 2; step > 0; step >>= 1)
      if (upto[at + step - 1] <= unit) at += step;
    chunk_join_unit<DIM>(p, all[at], unit - (at > 0 ? upto[at - 1] : 0), units_of(all[at], 0), share_o, share_ml);
  }
}

static bool mult8(int64_t x) { return (x & 7) == 0; }

static int chunk_pairs() { return min(sm_count() / 2, CJ_MAX_CUTS + 1); }

template <int DIM>
static int launch_chunk(const ChunkParams& p, const CUtensorMap& map_q, const CUtensorMap& map_k, const CUtensorMap& map_v, cudaStream_t stream) {
  const auto kernel = p.gate ? chunk_pair_kernel<DIM, true> : chunk_pair_kernel<DIM, false>;
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    for (const auto k : {chunk_pair_kernel<DIM, true>, chunk_pair_kernel<DIM, false>}) {
      if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, ChunkShape<DIM>::SMEM) != cudaSuccess)
        return fail(ERR_RUNTIME, "paged_gqa_attention_chunk: cannot raise dynamic shared memory to %d", ChunkShape<DIM>::SMEM);
      cudaFuncAttributes attr;  // its warpgroups exchange registers: with fewer at the launch than they share out they would wait for good
      if (cudaFuncGetAttributes(&attr, k) != cudaSuccess || attr.numRegs != CA_REGS)
        return fail(ERR_RUNTIME, "paged_gqa_attention_chunk: the kernel was not built with %d registers per thread", CA_REGS);
    }
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int pairs = chunk_pairs();
  if (launch_pdl_cluster(false, 2, kernel, dim3(2 * pairs), dim3(CA_THREADS), ChunkShape<DIM>::SMEM, stream, map_q, map_k, map_v, p) != cudaSuccess)
    return fail(ERR_LAUNCH, "paged_gqa_attention_chunk: %s", cudaGetErrorString(cudaGetLastError()));
  if (pairs > 1 && launch_pdl(true, chunk_join_kernel<DIM>, dim3(CJ_GRID * sm_count()), dim3(CJ_THREADS), 0, stream, p, pairs - 1) != cudaSuccess)
    return fail(ERR_LAUNCH, "paged_gqa_attention_chunk: %s", cudaGetErrorString(cudaGetLastError()));
  return check_launch("paged_gqa_attention_chunk");
}

}  // namespace b200

using namespace b200;

extern "C" int64_t b200_paged_gqa_attention_chunk_workspace_bytes(int32_t head_dim) {
  const int64_t pairs = static_cast<int64_t>(chunk_pairs()) * (2 * 256 * (head_dim + 2) * sizeof(float) + sizeof(ChunkCut));
  const int64_t few = chunk_few_workspace_bytes(head_dim);
  return pairs > few ? pairs : few;
}

extern "C" int b200_paged_gqa_attention_chunk(const b200_chunk_attention_args* args, b200_stream_t stream) {
  const b200_chunk_attention_args& a = *args;
  constexpr int64_t most = 0x7fffffff;
  B200_REQUIRE(a.batch > 0 && a.batch < most && a.total_tokens >= 0 && a.total_tokens <= most && a.num_pages > 0 && a.num_pages <= most &&
                   a.max_pages > 0 && a.max_pages <= most,
               "paged_gqa_attention_chunk: empty shape, or more than 2^31 of something");
  B200_REQUIRE(a.head_dim == 128 || a.head_dim == 256, "paged_gqa_attention_chunk: head_dim must be 128 or 256 (got %lld)",
               static_cast<long long>(a.head_dim));
  B200_REQUIRE(a.num_kv_heads > 0 && a.num_kv_heads <= 1024 && a.num_q_heads > 0 && a.num_q_heads % a.num_kv_heads == 0 &&
                   a.num_q_heads / a.num_kv_heads <= 64,
               "paged_gqa_attention_chunk: needs 1 to 64 Q heads per KV head, of which 1024 at most (got %lld/%lld)",
               static_cast<long long>(a.num_q_heads), static_cast<long long>(a.num_kv_heads));
  B200_REQUIRE(aligned16(a.q) && aligned16(a.k_cache) && aligned16(a.v_cache) && aligned16(a.out) && aligned16(a.gate) && mult8(a.q_stride_t) &&
                   mult8(a.q_stride_h) && mult8(a.kc_stride_p) && mult8(a.kc_stride_h) && mult8(a.kc_stride_s) && mult8(a.vc_stride_p) &&
                   mult8(a.vc_stride_h) && mult8(a.vc_stride_s) && mult8(a.gate_stride_t) && mult8(a.out_stride_t),
               "paged_gqa_attention_chunk: tensors must be 16-byte aligned with strides that are multiples of 8");
  const int dim = static_cast<int>(a.head_dim);
  const int64_t need = b200_paged_gqa_attention_chunk_workspace_bytes(dim);
  B200_REQUIRE(a.workspace_bytes >= need && a.workspace != nullptr && aligned16(a.workspace),
               "paged_gqa_attention_chunk: needs a 16-byte aligned workspace of %lld bytes", static_cast<long long>(need));
  if (a.total_tokens == 0) return OK;
  ChunkParams p = {};
  p.gate = static_cast<const __nv_bfloat16*>(a.gate);
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.bt_b = a.bt_stride_b, p.gate_t = a.gate_stride_t, p.out_t = a.out_stride_t;
  p.block_table = a.block_table, p.cu_seqlens = a.cu_seqlens, p.pos = a.pos;
  p.batch = a.batch, p.tokens = a.total_tokens, p.num_pages = a.num_pages, p.max_pages = a.max_pages;
  p.hkv = a.num_kv_heads, p.group = a.num_q_heads / a.num_kv_heads;
  p.scale_log2 = 1.4426950408889634f / sqrtf(static_cast<float>(dim));
  p.err = wait_timeout_flag();
  if (!p.err) return fail(ERR_RUNTIME, "paged_gqa_attention_chunk: no error flag");
  const auto st = reinterpret_cast<cudaStream_t>(stream);
  if (chunk_takes_few(p.batch, p.tokens, p.hkv, p.group)) return launch_chunk_few(p, a, st);
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = p.part_o + static_cast<int64_t>(chunk_pairs()) * 2 * 256 * dim;
  p.cuts = reinterpret_cast<ChunkCut*>(p.part_ml + static_cast<int64_t>(chunk_pairs()) * 2 * 256 * 2);
  const int per_cta = 128 / p.group;
  p.per = 2 * per_cta, p.gap = CA_GAP, p.least = CA_MIN_SHARE, p.whole = (p.tokens / p.per + p.batch) * p.hkv < chunk_pairs() ? CA_WHOLE_FEW : CA_WHOLE;
  CUtensorMap map_q, map_k, map_v;
  // q as {64 columns, heads of a group, groups, tokens, column blocks}; one load = a CTA's tokens of one group, one block
  const uint64_t dims[5] = {64, static_cast<uint64_t>(p.group), static_cast<uint64_t>(p.hkv), static_cast<uint64_t>(p.tokens),
                            static_cast<uint64_t>(dim / 64)};
  const uint64_t strides[4] = {static_cast<uint64_t>(a.q_stride_h) * 2, static_cast<uint64_t>(a.q_stride_h) * 2 * p.group,
                               static_cast<uint64_t>(a.q_stride_t) * 2, 128};
  const uint32_t box[5] = {64, static_cast<uint32_t>(p.group), 1, static_cast<uint32_t>(per_cta), 1};
  if (!encode_map_bf16_sw128(&map_q, a.q, 5, dims, strides, box) ||
      !encode_pages(&map_k, a.k_cache, dim, p.hkv, p.num_pages, a.kc_stride_p, a.kc_stride_h, a.kc_stride_s, 8, dim / 64) ||
      !encode_pages(&map_v, a.v_cache, dim, p.hkv, p.num_pages, a.vc_stride_p, a.vc_stride_h, a.vc_stride_s, PAGE, dim / 128))
    return fail(ERR_RUNTIME, "paged_gqa_attention_chunk: cannot encode the tensor maps of q and the pools");
  return dim == 256 ? launch_chunk<256>(p, map_q, map_k, map_v, st) : launch_chunk<128>(p, map_q, map_k, map_v, st);
}
