// Attention of new tokens over the paged cache (see chunk_attention.cu) for calls of few tokens per sequence, bound by the bytes of the cache:
// a decode step, the check of a speculated continuation.
//
// A block is up to 8 NT query rows of a key/value head (row = token * G + head).  Its pages are the unit of work: one warp, one page,
// keys as the M dimension of the warp's matrix products, so that few rows cost a narrow N instead of a wide M:
//     S^T[16 x 8 NT]  = K_page[16 x D] . Q^T[D x 8 NT]              mma.sync m16n8k16, Q^T from shared memory
//     O^T[D x 8 NT]  += V_page^T[D x 16] . P^T[16 x 8 NT]           P in bf16, as V is (both operands have one type): 2^-8 of itself at
//                                                                   most; its sum stays in fp32
// (tcgen05 wants 128 rows, of which 16 would be used; 32 NT small products a page take less than a tenth of the page's time on the bus.)
// The line of all blocks' pages is cut evenly over one CTA per SM, as in chunk_attention.cu; the eight warps of a CTA take the pages of a
// piece in turn, each with a K and a V page of its own on their way (128-byte swizzle, one box per page), the next piece's first pages
// before this one's end.  At a piece's end the warps' states are merged in shared memory.  A block cut between CTAs leaves one partial per
// CTA, and a second kernel joins them in the order of the keys.  (By the last CTA to arrive, which the first version did, 4 rows over 32 000 keys
// take 26 us, so 18; 8 rows 40 and 19; nowhere less.)
// Slots of the last page behind the block's end are cleared in shared memory, for zeros of P do not help against NaN in V.  (An infinity or
// NaN among the values of a block's own tokens does make the rows in front of it NaN, whose P is zero there.)
// Every wait is bounded; a CTA that gives up sets the device error flag.
// Bound by the cache's bytes: 4 x 1 tokens over 30 000 to 32 767, 8 + 2 heads of 256 (251 MB), 46 us, 5.5 TB/s of 6.5; 32 x 4 over 512 to
// 4092 (144 MB) 38 us, of which the join is 5.5, launch, lengths, tables and first pages some 6; one token over 10 8.
#include "chunk.cuh"

namespace b200 {

constexpr int CF_WARPS = 8, CF_THREADS = CF_WARPS * 32;
constexpr int CF_ROWS = 16;                          // most rows of a block
constexpr int CF_SLOTS = 4;                          // warps that merge at a time
constexpr int CF_GAP = 24 * PAGE;                    // what a block costs once, in keys: 8 x 4 tokens over 4000 23.4 us, 8 pages: 26.5, 48: 24.1
constexpr int CF_LEAST = 8 * PAGE;                   // least stretch of the line for a CTA, a page a warp: 1 x 4 over 500 13.0 us, 16: 14.5, 32: 18.5

template <int DIM, int NT>
struct FewShape {
  static constexpr int ROWS = 8 * NT, TILE = PAGE * DIM * 2, Q_PITCH = DIM * 2 + 16;  // bytes
  static constexpr int ACC_PITCH = DIM + 4;                                          // floats: no bank conflicts
  static constexpr int RING = CF_WARPS * 2 * TILE, Q = 2 * ROWS * Q_PITCH, MERGE = CF_SLOTS * ROWS * ACC_PITCH * 4;
  static constexpr int SMEM = RING + Q + MERGE;
};

// 16-byte piece `chunk` of row `row` in a page that the copy engine brought as {64 columns, 16 slots, D/64 blocks} with the 128-byte swizzle
__device__ __forceinline__ uint32_t page_offset(int row, int chunk) {
  return static_cast<uint32_t>((chunk >> 3) * (PAGE * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// Four dimensions of a block's row n: divided, gated, stored.
template <int DIM>
__device__ __forceinline__ void few_finish(const ChunkParams& p, int row0, int h, int n, int d, float4 v, float sum) {
  const int tok = n / p.group;
  const int64_t t = row0 + tok, col = static_cast<int64_t>(h * p.group + n - tok * p.group) * DIM + d;
  const float inv = 1.f / sum;
  uint64_t v0 = f32x2(v.x * inv, v.y * inv), v1 = f32x2(v.z * inv, v.w * inv);
  if (p.gate) {
    const uint2 g = *reinterpret_cast<const uint2*>(p.gate + t * p.gate_t + col);
    v0 = gate_pair(v0, g.x), v1 = gate_pair(v1, g.y);
  }
  *reinterpret_cast<uint2*>(p.out + t * p.out_t + col) = make_uint2(pack_bf16x2(v0), pack_bf16x2(v1));
}

template <int DIM, int NT>
__global__ void __launch_bounds__(CF_THREADS, 1)
chunk_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ ChunkParams p,
                 const __nv_bfloat16* q, int64_t q_t, int64_t q_h) {
  using Shape = FewShape<DIM, NT>;
  constexpr int ROWS = Shape::ROWS, TILE = Shape::TILE;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t bars[CF_WARPS][2];
  __shared__ float s_ml[CF_WARPS][2][ROWS];          // the warps' maxima and sums
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* tiles = smem + warp * 2 * TILE;           // K, V
  uint8_t* q_s = smem + Shape::RING;
  float* merge = reinterpret_cast<float*>(q_s + Shape::Q);
  if (lane == 0) {
    mbar_init(&bars[warp][0], 1);
    mbar_init(&bars[warp][1], 1);
    mbar_fence_init();
    if (warp == 0) {
      prefetch_tensormap(&map_k);
      prefetch_tensormap(&map_v);
    }
  }
  __syncwarp();
  pdl_trigger();                                     // (the second kernel waits for this grid before it reads anything)
  if (tid == 0) p.cuts[2 * blockIdx.x] = p.cuts[2 * blockIdx.x + 1] = ChunkCut{};
  // ---- this CTA's stretch; every warp walks along it by itself
  const int parts = gridDim.x, me = blockIdx.x;
  const int per_lane = (p.batch + 31) / 32;
  int64_t in_front, mine;
  const int64_t line = chunk_line(p, lane, per_lane, in_front, mine), share = chunk_share(p, line, parts);
  const int64_t from = me * share, to = min(line, from + share);
  if (from >= line) return;
  struct Piece {
    ChunkRow row;
    int t0, t1, all;  // its pages, those of the block
  };
  auto settle = [&](Piece& x) {  // the first piece from x.row on that has pages; none: x.t1 = x.t0
    x.t0 = x.t1 = 0;
    while (x.row.b < p.batch && x.row.at < to) {
      x.all = (x.row.keys(p) + PAGE - 1) / PAGE;
      x.t0 = x.row.cut<PAGE>(p, from, x.all);
      x.t1 = x.row.cut<PAGE>(p, to, x.all);
      if (x.t1 > x.t0) return;
      chunk_next(p, x.row);
    }
    x.t1 = x.t0;
  };
  // ---- pages on their way: `ahead` is the piece whose pages are asked for, up to `asked`; ids of 32 of the warp's pages at a time
  Piece now, ahead;
  now.row = chunk_find(p, from, lane, per_lane, in_front, mine);
  settle(now);
  if (now.t1 <= now.t0) return;
  ahead = now;
  int asked = 0, ids = 0;
  bool more = true, dead = false;
  uint32_t phases = 0;
  auto load_ids = [&]() {
    const int lp = ahead.t0 + warp + CF_WARPS * (asked + lane);
    int id = -1;
    if (lp < ahead.t1 && lp < p.max_pages) id = p.block_table[ahead.row.b * p.bt_b + lp];
    ids = id >= 0 && id < p.num_pages ? id : -1;  // (-1: a box outside the pool, zeros)
  };
  load_ids();
  // the next page's K or V; both take the same page, K first
  auto ask = [&](int which) {
    const int id = __shfl_sync(0xffffffffu, ids, asked & 31);
    if (!more || dead) return;
    if (lane == 0) {
      mbar_expect_tx(&bars[warp][which], TILE);
      tma_load_5d(tiles + which * TILE, which ? &map_v : &map_k, 0, 0, 0, ahead.row.h, id, &bars[warp][which]);
    }
  };
  // to the warp's next page: of this piece, of the next one that has any for it
  auto advance = [&]() {
    ++asked;
    while (more && ahead.t0 + warp + CF_WARPS * asked >= ahead.t1) {
      chunk_next(p, ahead.row);
      settle(ahead);
      asked = 0;
      more = ahead.t1 > ahead.t0;
      if (more && ahead.t0 + warp < ahead.t1) {
        load_ids();
        return;
      }
    }
    if (more && (asked & 31) == 0) load_ids();
  };
  if (ahead.t0 + warp >= ahead.t1) asked = -1, advance();
  ask(0);
  ask(1);
  // ---- queries of a piece, rows behind its last token as zeros
  auto stage_q = [&](const Piece& x, int buf) {
    const int first = x.row.j * p.per, rows = min(p.per, x.row.q.n - first) * p.group;
    for (int i = tid; i < ROWS * (DIM / 8); i += CF_THREADS) {
      const int r = i / (DIM / 8), c = i % (DIM / 8), tok = r / p.group;
      uint8_t* dst = q_s + buf * (ROWS * Shape::Q_PITCH) + r * Shape::Q_PITCH + c * 16;
      if (r < rows) cp_async16(dst, q + (x.row.q.start + first + tok) * q_t + (x.row.h * p.group + r - tok * p.group) * q_h + c * 8);
      else *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
    }
    cp_async_commit();
  };
  stage_q(now, 0);
  cp_async_wait_all();
  __syncthreads();

  const float scale = p.scale_log2;
  const uint32_t k_tile = smem_u32(tiles), v_tile = k_tile + TILE;
  for (int piece = 0; now.t1 > now.t0; ++piece) {
    Piece next = now;
    chunk_next(p, next.row);
    settle(next);
    if (next.t1 > next.t0) stage_q(next, (piece + 1) & 1);
    const int first = now.row.j * p.per, count = min(p.per, now.row.q.n - first), rows = count * p.group;
    const int key0 = now.row.q.s + first, keys = now.row.keys(p);  // the last key that the first token sees; keys of the last token
    const uint32_t q_addr = smem_u32(q_s) + (piece & 1) * (ROWS * Shape::Q_PITCH);
    float o[DIM / 16][NT][4], m[NT][2], l[NT][2];
    int lim[NT][2];  // last key that a column's row sees
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < DIM / 16; ++i) o[i][t][0] = o[i][t][1] = o[i][t][2] = o[i][t][3] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[t][c] = -INFINITY, l[t][c] = 0.f;
        lim[t][c] = min(key0 + min((t * 8 + (lane & 3) * 2 + c) / p.group, count - 1), keys - 1);
      }
    }
    for (int page = now.t0 + warp; page < now.t1; page += CF_WARPS) {
      // ---- scores of a page
      if (!dead) dead = !warp_wait_bounded(&bars[warp][0], phases & 1);
      phases ^= 1;
      float s[NT][4] = {}, s2[NT][4] = {};
      {
        const int row = (lane & 7) + ((lane >> 3) & 1) * 8, col = lane >> 4;  // of the K page
        const uint32_t q_row = NT == 2 ? q_addr + ((lane & 7) + (lane >> 4) * 8) * Shape::Q_PITCH + ((lane >> 3) & 1) * 16
                                       : q_addr + (lane & 7) * Shape::Q_PITCH + (lane >> 3) * 16;
#pragma unroll
        for (int ks = 0; ks < DIM / 16; ks += 2) {
          uint32_t a0[4], a1[4], b[4], b2[4];
          ldmatrix_x4(a0, k_tile + page_offset(row, ks * 2 + col));
          ldmatrix_x4(a1, k_tile + page_offset(row, ks * 2 + 2 + col));
          ldmatrix_x4(b, q_row + ks * 32);
          if (NT == 2) {
            ldmatrix_x4(b2, q_row + ks * 32 + 32);
            mma_bf16_16816(s[0], a0, b[0], b[1]);
            mma_bf16_16816(s[NT - 1], a0, b[2], b[3]);
            mma_bf16_16816(s2[0], a1, b2[0], b2[1]);
            mma_bf16_16816(s2[NT - 1], a1, b2[2], b2[3]);
          } else {
            mma_bf16_16816(s[0], a0, b[0], b[1]);
            mma_bf16_16816(s2[0], a1, b[2], b[3]);
          }
        }
      }
      __syncwarp();
      advance();  // (`asked` was this page; its V is on its way)
      ask(0);
      const int key = page * PAGE + (lane >> 2);  // of the lane's first row, the second is 8 behind
      const bool edge = page * PAGE + PAGE - 1 > key0;
      uint32_t pb[NT][2];
      float alpha[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float x[4], mx[2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = (s[t][e] + s2[t][e]) * scale;
          if (edge && key + (e >> 1) * 8 > lim[t][e & 1]) x[e] = -INFINITY;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          mx[c] = fmaxf(x[c], x[c + 2]);
#pragma unroll
          for (int w = 4; w <= 16; w <<= 1) mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], w));
          const float m_new = fmaxf(m[t][c], mx[c]), at = m_new == -INFINITY ? 0.f : m_new;  // (a row that has seen nothing yet)
          alpha[t][c] = ex2_fast(m[t][c] - at);
          x[c] = ex2_fast(x[c] - at), x[c + 2] = ex2_fast(x[c + 2] - at);
          l[t][c] = l[t][c] * alpha[t][c] + (x[c] + x[c + 2]);
          m[t][c] = m_new;
        }
        pb[t][0] = movmatrix_trans(pack_bf16(x[0], x[1]));
        pb[t][1] = movmatrix_trans(pack_bf16(x[2], x[3]));
      }
      bool rescale = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) rescale |= alpha[t][0] != 1.f || alpha[t][1] != 1.f;
      if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
        for (int i = 0; i < DIM / 16; ++i)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][t][e] *= alpha[t][e & 1];
      }
      // ---- values
      if (!dead) dead = !warp_wait_bounded(&bars[warp][1], (phases >> 1) & 1);
      phases ^= 2;
      const int valid = keys - page * PAGE;
      if (valid < PAGE) {
        for (int i = lane; i < (PAGE - valid) * (DIM / 8); i += 32)
          *reinterpret_cast<uint4*>(tiles + TILE + page_offset(valid + i / (DIM / 8), i % (DIM / 8))) = make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
      {
        const int row = (lane & 7) + (lane >> 4) * 8, col = (lane >> 3) & 1;
#pragma unroll
        for (int i = 0; i < DIM / 16; ++i) {
          uint32_t a[4];
          ldmatrix_x4_trans(a, v_tile + page_offset(row, i * 2 + col));
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_bf16_16816(o[i][t], a, pb[t][0], pb[t][1]);
        }
      }
      if (valid < PAGE) fence_proxy_async();  // the cleared rows in front of the next copy
      __syncwarp();
      ask(1);
    }
    // ---- merge the eight warps
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int w = 4; w <= 16; w <<= 1) l[t][c] += __shfl_xor_sync(0xffffffffu, l[t][c], w);
        if (lane < 4) {
          s_ml[warp][0][t * 8 + lane * 2 + c] = m[t][c];
          s_ml[warp][1][t * 8 + lane * 2 + c] = l[t][c];
        }
      }
    auto put = [&]() {
      float* to_s = merge + (warp % CF_SLOTS) * ROWS * Shape::ACC_PITCH + (lane >> 2);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < DIM / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) to_s[(t * 8 + (lane & 3) * 2 + (e & 1)) * Shape::ACC_PITCH + i * 16 + (e >> 1) * 8] = o[i][t][e];
    };
    if (warp < CF_SLOTS) put();
    __syncthreads();
    constexpr int QUADS = DIM / 4, MINE = ROWS * QUADS / CF_THREADS > 0 ? ROWS * QUADS / CF_THREADS : 1;  // of this thread: 4 dimensions of a row each
    float4 acc[MINE];
    float m_all[MINE], l_all[MINE];
#pragma unroll
    for (int k = 0; k < MINE; ++k) {
      const int n = (tid + k * CF_THREADS) / QUADS;
      float mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int w = 0; w < CF_WARPS; ++w) mm = fmaxf(mm, s_ml[w][0][n]);
#pragma unroll
      for (int w = 0; w < CF_WARPS; ++w)
        if (s_ml[w][0][n] != -INFINITY) ll += s_ml[w][1][n] * ex2_fast(s_ml[w][0][n] - mm);
      m_all[k] = mm, l_all[k] = ll, acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int half = 0; half < CF_WARPS / CF_SLOTS; ++half) {
      if (half > 0) {
        __syncthreads();
        if (warp >= CF_SLOTS) put();
        __syncthreads();
      }
#pragma unroll
      for (int k = 0; k < MINE; ++k) {
        const int i = tid + k * CF_THREADS, n = i / QUADS, d = (i % QUADS) * 4;
#pragma unroll
        for (int w = 0; w < CF_SLOTS; ++w) {
          const float mw = s_ml[half * CF_SLOTS + w][0][n];
          if (mw == -INFINITY) continue;  // the row sees nothing of that warp's pages
          const float f = ex2_fast(mw - m_all[k]);
          const float4 x = *reinterpret_cast<const float4*>(merge + (w * ROWS + n) * Shape::ACC_PITCH + d);
          acc[k].x = fmaf(x.x, f, acc[k].x), acc[k].y = fmaf(x.y, f, acc[k].y);
          acc[k].z = fmaf(x.z, f, acc[k].z), acc[k].w = fmaf(x.w, f, acc[k].w);
        }
      }
    }
    auto finish = [&](int i, float4 v, float sum) { few_finish<DIM>(p, now.row.q.start + first, now.row.h, i / QUADS, (i % QUADS) * 4, v, sum); };
    if (now.t0 == 0 && now.t1 == now.all) {
#pragma unroll
      for (int k = 0; k < MINE; ++k)
        if (tid + k * CF_THREADS < rows * QUADS) finish(tid + k * CF_THREADS, acc[k], l_all[k]);
    } else {
      // ---- a partial, for the second kernel to join
      const int begins = static_cast<int>(now.row.at / share), last = now.row.last_stretch<PAGE>(p, share, now.all);
      const int begin = now.row.first_stretch<PAGE>(p, share, now.all);
      auto slot_of = [&](int i) { return static_cast<int64_t>(2 * i + (i == begins)); };
#pragma unroll
      for (int k = 0; k < MINE; ++k) {
        const int i = tid + k * CF_THREADS, n = i / QUADS;
        if (i >= rows * QUADS) continue;
        *reinterpret_cast<float4*>(p.part_o + slot_of(me) * (CF_ROWS * DIM) + i * 4) = acc[k];
        if (i % QUADS == 0) reinterpret_cast<float2*>(p.part_ml)[slot_of(me) * CF_ROWS + n] = make_float2(m_all[k], l_all[k]);
      }
      if (me == begin && tid == 0) {
        ChunkCut cut = {};
        cut.row0 = now.row.q.start + first, cut.count = count, cut.h = now.row.h;
        cut.first = begins, cut.begin = begin, cut.last = last;
        p.cuts[slot_of(me)] = cut;
      }
    }
    now = next;
    cp_async_wait_all();
    __syncthreads();  // queries of the next piece are there, the merge buffers and sums free again
  }
  if (dead) {
    if (lane == 0) atomicExch(p.err, 1);
    for (int i = 0; i < 2; ++i) mbar_wait_bounded(&bars[warp][i], (phases >> i) & 1, 1u << 12);  // copies in flight
  }
}

// Joins the partial sums of cut blocks: grid (slots, CTAs of 64 groups of 4 dimensions of a row), a quarter of the pieces to a thread.
// Bound by launch, cuts and one round of loads.  (With the units counted first, as in chunk_attention.cu, 32 x 4 tokens over 2000 took 39.6 us,
// so 36.)
constexpr int CJ_QUADS = 64, CJ_SHARES = CF_THREADS / CJ_QUADS;
template <int DIM>
__global__ void __launch_bounds__(CF_THREADS)
chunk_few_join_kernel(const __grid_constant__ ChunkParams p) {
  __shared__ float4 part_o[CJ_SHARES][CJ_QUADS];
  __shared__ float2 part_ml[CJ_SHARES][CJ_QUADS];
  constexpr int QUADS = DIM / 4, AT_ONCE = 3;
  pdl_wait();
  const ChunkCut cut = p.cuts[blockIdx.x];
  const int tid = threadIdx.x, share = tid / CJ_QUADS, i = blockIdx.y * CJ_QUADS + tid % CJ_QUADS, n = i / QUADS, d = (i % QUADS) * 4;
  if (cut.last <= cut.begin || blockIdx.y * CJ_QUADS >= cut.count * p.group * QUADS) return;
  auto slot_of = [&](int c) { return static_cast<int64_t>(2 * c + (c == cut.first)); };
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto take = [&](float mi, float li, const float4& y) {
    if (mi == -INFINITY) return;  // the row sees nothing of this piece
    const float to = fmaxf(m, mi), f = ex2_fast(m - to), g = ex2_fast(mi - to);
    l = fmaf(l, f, li * g), m = to;
    o.x = fmaf(o.x, f, y.x * g), o.y = fmaf(o.y, f, y.y * g), o.z = fmaf(o.z, f, y.z * g), o.w = fmaf(o.w, f, y.w * g);
  };
#pragma unroll 1
  for (int c = cut.begin + share; c <= cut.last; c += CJ_SHARES * AT_ONCE) {  // a batch is asked for before any of it is used
    float2 x[AT_ONCE];
    float4 y[AT_ONCE];
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const int piece = c + k * CJ_SHARES;
      x[k] = make_float2(-INFINITY, 0.f);
      if (piece > cut.last) continue;
      x[k] = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + slot_of(piece) * CF_ROWS + n);
      y[k] = __ldcg(reinterpret_cast<const float4*>(p.part_o + slot_of(piece) * (CF_ROWS * DIM) + i * 4));
    }
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) take(x[k].x, x[k].y, y[k]);
  }
  part_o[share][tid % CJ_QUADS] = o;
  part_ml[share][tid % CJ_QUADS] = make_float2(m, l);
  __syncthreads();
  if (share > 0 || n >= cut.count * p.group) return;
#pragma unroll
  for (int c = 1; c < CJ_SHARES; ++c) take(part_ml[c][tid].x, part_ml[c][tid].y, part_o[c][tid]);
  few_finish<DIM>(p, cut.row0, cut.h, n, d, o, l);
}

// Calls whose blocks of 16 rows are mostly one per sequence and head, or two where half as many pairs of CTAs are not yet busy with a block each.
// us here and on pairs: 32 sequences of 16 rows over 2000 keys (2 heads of 256) 35, 53, one over 500 13.0, 15.0; of 32 rows: 32 sequences over
// 2000 44, 54, 8 over 4000 29, 32, but 64 over 4000 170, 129; 8 of 48 rows over 2000 24.5, 24.9, 16 of them 36, 33.
// The mean is all that the host knows: 63 single tokens beside a portion of 190 over 2000 61, 78; but 1000 tokens beside 255 idle sequences
// over 2000 151, 61, over 30 000 1098, 227, for each block of 16 rows reads the sequence again, where pairs take 256 at a time.
bool chunk_takes_few(int batch, int tokens, int hkv, int group) {
  const int blocks = static_cast<int64_t>(batch) * hkv * 2 <= sm_count() ? 2 : 1;
  return group <= CF_ROWS && static_cast<int64_t>(tokens) * group <= static_cast<int64_t>(batch) * (CF_ROWS * blocks);
}

int64_t chunk_few_workspace_bytes(int dim) {
  return static_cast<int64_t>(sm_count()) * 2 * (CF_ROWS * (dim + 2) * sizeof(float) + sizeof(ChunkCut));
}

template <int DIM, int NT>
static int launch_few(const ChunkParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v, const b200_chunk_attention_args& a, cudaStream_t stream) {
  constexpr int smem = FewShape<DIM, NT>::SMEM;
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (cudaFuncSetAttribute(chunk_few_kernel<DIM, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return fail(ERR_RUNTIME, "paged_gqa_attention_chunk: cannot raise dynamic shared memory to %d", smem);
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int parts = sm_count(), rows = min(p.per, p.tokens) * p.group;
  chunk_few_kernel<DIM, NT><<<parts, CF_THREADS, smem, stream>>>(map_k, map_v, p, static_cast<const __nv_bfloat16*>(a.q), a.q_stride_t, a.q_stride_h);
  if (launch_pdl(true, chunk_few_join_kernel<DIM>, dim3(2 * parts, (rows * (DIM / 4) + CJ_QUADS - 1) / CJ_QUADS), dim3(CF_THREADS), 0, stream, p) !=
      cudaSuccess)
    return fail(ERR_LAUNCH, "paged_gqa_attention_chunk: %s", cudaGetErrorString(cudaGetLastError()));
  return check_launch("paged_gqa_attention_chunk");
}

int launch_chunk_few(ChunkParams p, const b200_chunk_attention_args& a, cudaStream_t stream) {
  const int dim = static_cast<int>(a.head_dim);
  // (half the products for blocks of 8 rows: 32 x 2 tokens over 2000 32.2 us, so 34.5 by blocks of 16; 32 x 1 29.8, 33.5)
  const bool narrow = p.group <= 8 && static_cast<int64_t>(p.tokens) * p.group <= static_cast<int64_t>(p.batch) * 8;
  p.per = (narrow ? 8 : 16) / p.group, p.gap = CF_GAP, p.least = CF_LEAST, p.whole = 0;
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = p.part_o + static_cast<int64_t>(sm_count()) * 2 * CF_ROWS * dim;
  p.cuts = reinterpret_cast<ChunkCut*>(p.part_ml + static_cast<int64_t>(sm_count()) * 2 * CF_ROWS * 2);
  CUtensorMap map_k, map_v;
  if (!encode_pages(&map_k, a.k_cache, dim, p.hkv, p.num_pages, a.kc_stride_p, a.kc_stride_h, a.kc_stride_s, PAGE, dim / 64) ||
      !encode_pages(&map_v, a.v_cache, dim, p.hkv, p.num_pages, a.vc_stride_p, a.vc_stride_h, a.vc_stride_s, PAGE, dim / 64))
    return fail(ERR_RUNTIME, "paged_gqa_attention_chunk: cannot encode the tensor maps of the pools");
  const auto launch = [&](auto form256, auto form128) { return (dim == 256 ? form256 : form128)(p, map_k, map_v, a, stream); };
  return narrow ? launch(launch_few<256, 1>, launch_few<128, 1>) : launch(launch_few<256, 2>, launch_few<128, 2>);
}

}  // namespace b200
