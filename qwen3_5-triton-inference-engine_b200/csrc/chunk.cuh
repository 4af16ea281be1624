// Attention of new tokens over the paged cache: what its two kernels share.  chunk_attention.cu: pairs of CTAs on tcgen05; chunk_few.cu: one CTA
// to an SM on blocks of up to 16 rows, for calls of few tokens per sequence.
#pragma once
#include "b200_attn.h"
#include "umma.cuh"

namespace b200 {

struct ChunkParams {
  const __nv_bfloat16* gate;
  __nv_bfloat16* out;
  int64_t bt_b, gate_t, out_t;
  const int32_t *block_table, *cu_seqlens;
  const int64_t* pos;
  float *part_o, *part_ml;  // pairs: [2 slots of each pair][D/4][256 rows][4], [slot][256 rows][2]; few: [2 slots of each CTA][16 rows][D], ...[2]
  struct ChunkCut* cuts;    // pairs: one each, of the row that begins in a pair's stretch and goes on behind it; few: at its first partial's slot
  int batch, tokens, num_pages, max_pages, hkv, group;
  int per;                  // query tokens of a block
  int gap;                  // what a block's row costs once, in keys
  int least;                // least stretch of the line for a CTA or pair, more than a tile or page
  int whole;                // rows up to this long are not cut
  float scale_log2;
  int* err;
};

// o sigmoid(g) for two values at a time: with e = 2^(-|g| log2 e), which is at most 1, sigmoid(g) = (g < 0 ? e : 1) / (1 + e), and 1 / (1 + e) is
// a polynomial (Chebyshev interpolation of degree 5 on [0, 1], off by 2^-14.2 of itself).  One exponential per value; by expf and a division the
// output warps of chunk_attention.cu take three times as long.
__device__ __forceinline__ uint64_t gate_pair(uint64_t o, uint32_t g) {
  const float a = bf16_lo(g), b = bf16_hi(g), ea = ex2_fast(fabsf(a) * -1.4426950408889634f), eb = ex2_fast(fabsf(b) * -1.4426950408889634f);
  const uint64_t e = f32x2(ea, eb);
  uint64_t r = f32x2_fma(e, f32x2(-0.10448446869850159f, -0.10448446869850159f), f32x2(0.41793787479400635f, 0.41793787479400635f));
  r = f32x2_fma(r, e, f32x2(-0.7705729007720947f, -0.7705729007720947f));
  r = f32x2_fma(r, e, f32x2(0.9534207582473755f, 0.9534207582473755f));
  r = f32x2_fma(r, e, f32x2(-0.9962757229804993f, -0.9962757229804993f));
  r = f32x2_fma(r, e, f32x2(0.9999489784240723f, 0.9999489784240723f));
  return f32x2_mul(f32x2_mul(o, f32x2(a < 0.f ? ea : 1.f, b < 0.f ? eb : 1.f)), r);
}

// ----------------------------------------------------------------------------- the line
// A sequence's place in it: new tokens n from packed row `start`, s tokens held in front of them.
struct ChunkSeq {
  int start, n, s;
};
__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkParams& p, int b) {
  ChunkSeq q;
  const int from = p.cu_seqlens[b], to = min(p.cu_seqlens[b + 1], p.tokens);
  q.start = max(from, 0);
  q.n = max(to - q.start, 0);
  // (a sequence that begins in front of the packed rows: its tokens there are as good as held)
  const int64_t most = min(static_cast<int64_t>(p.max_pages) * PAGE, static_cast<int64_t>(1) << 30) - 1;
  const int64_t held = min(max(p.pos[b], static_cast<int64_t>(0)), most) + (q.start - static_cast<int64_t>(from));
  q.s = static_cast<int>(min(held, most));
  return q;
}
// Length of the first j blocks of one head, all of them whole; j below the number of blocks.
__device__ __forceinline__ int64_t chunk_before(const ChunkParams& p, const ChunkSeq& q, int64_t j) {
  return j * (q.s + p.gap) + p.per * (j * (j + 1) / 2);
}
__device__ __forceinline__ int64_t chunk_head(const ChunkParams& p, const ChunkSeq& q) {  // of one head
  const int blocks = (q.n + p.per - 1) / p.per;
  return blocks == 0 ? 0 : chunk_before(p, q, blocks - 1) + q.s + q.n + p.gap;
}

struct ChunkRow {
  int b, h, j;
  ChunkSeq q;
  int64_t at, length;  // place on the line
  __device__ __forceinline__ int keys(const ChunkParams& p) const {  // that the block's last token sees
    const int per = p.per;
    const int64_t k = q.s + min(static_cast<int64_t>(j + 1) * per, static_cast<int64_t>(q.n));
    return static_cast<int>(min(k, static_cast<int64_t>(p.max_pages) * PAGE));
  }
  // tiles of TILE keys in front of place x of the line; a short row is in front of it or behind it as a whole
  template <int TILE>
  __device__ __forceinline__ int cut(const ChunkParams& p, int64_t x, int tiles) const {
    if (x <= at) return 0;
    if (x >= at + length) return tiles;
    if (length <= p.whole) return x > at + length / 2 ? tiles : 0;
    return static_cast<int>(min((x - at + TILE / 2) / TILE, static_cast<int64_t>(tiles)));
  }
  // the first and the last stretch of `share` that have any of them (all of them: `tiles`).  A stretch is longer than a tile, so that only
  // the row's first one, and what follows its last tile, may have none
  template <int TILE>
  __device__ __forceinline__ int first_stretch(const ChunkParams& p, int64_t share, int tiles) const {
    if (length <= p.whole) return static_cast<int>((at + length / 2) / share);
    const int begins = static_cast<int>(at / share);
    return cut<TILE>(p, (begins + 1) * share, tiles) > 0 ? begins : begins + 1;
  }
  template <int TILE>
  __device__ __forceinline__ int last_stretch(const ChunkParams& p, int64_t share, int tiles) const {
    if (length <= p.whole) return static_cast<int>((at + length / 2) / share);
    return static_cast<int>((at + static_cast<int64_t>(tiles) * TILE - TILE / 2 - 1) / share);
  }
};

// What joins the partial sums of a cut row has to know: they lie with the parts of the line from `begin` to `last`, in the second slot of
// `first`, where it begins, and in the first slot of the others.
struct ChunkCut {
  int row0, count, h;       // packed row of its first token, its tokens, kv head
  int first, begin, last;   // no more than one piece: nothing to join
  int pad[2];
};

__device__ __forceinline__ int64_t warp_prefix(int64_t v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}
// The whole line, and for a lane the length in front of its part of the sequences.
__device__ __forceinline__ int64_t chunk_line(const ChunkParams& p, int lane, int per_lane, int64_t& in_front, int64_t& mine) {
  mine = 0;
  for (int i = 0; i < per_lane; ++i) {
    const int b = lane * per_lane + i;
    if (b < p.batch) mine += chunk_head(p, chunk_seq(p, b)) * p.hkv;
  }
  const int64_t upto = warp_prefix(mine, lane);
  in_front = upto - mine;
  return __shfl_sync(0xffffffffu, upto, 31);
}
// The row that place x (inside the line) falls into; the whole warp.
__device__ __forceinline__ ChunkRow chunk_find(const ChunkParams& p, int64_t x, int lane, int per_lane, int64_t in_front, int64_t mine) {
  const int owner = __ffs(__ballot_sync(0xffffffffu, x >= in_front && x < in_front + mine)) - 1;
  int64_t at = __shfl_sync(0xffffffffu, in_front, owner);
  ChunkRow r;
  const int end = min((owner + 1) * per_lane, p.batch);
  for (int b0 = owner * per_lane; b0 < end; b0 += 32) {
    ChunkSeq q = {0, 0, 0};
    int64_t len = 0;
    if (b0 + lane < end) {
      q = chunk_seq(p, b0 + lane);
      len = chunk_head(p, q) * p.hkv;
    }
    const int64_t upto = warp_prefix(len, lane);
    const uint32_t has = __ballot_sync(0xffffffffu, at + upto > x);
    if (has == 0) {
      at += __shfl_sync(0xffffffffu, upto, 31);
      continue;
    }
    const int src = __ffs(has) - 1;
    r.b = b0 + src;
    r.q.start = __shfl_sync(0xffffffffu, q.start, src);
    r.q.n = __shfl_sync(0xffffffffu, q.n, src);
    r.q.s = __shfl_sync(0xffffffffu, q.s, src);
    at += __shfl_sync(0xffffffffu, upto - len, src);
    break;
  }
  const int per = p.per;
  const int64_t head = chunk_head(p, r.q);
  r.h = static_cast<int>((x - at) / head);
  at += r.h * head;
  int low = 0, high = (r.q.n + per - 1) / per;  // before(low) <= x - at < before(high)
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (chunk_before(p, r.q, mid) <= x - at) low = mid;
    else high = mid;
  }
  r.j = low;
  r.at = at + chunk_before(p, r.q, low);
  r.length = r.q.s + min((low + 1) * per, r.q.n) + p.gap;
  return r;
}
// The row behind r (b = batch: none); uniform.
__device__ __forceinline__ void chunk_next(const ChunkParams& p, ChunkRow& r) {
  const int per = p.per;
  r.at += r.length;
  ++r.j;
  if (r.j * per >= r.q.n) {
    r.j = 0;
    if (++r.h == p.hkv) {
      r.h = 0;
      do {
        if (++r.b >= p.batch) return;
        r.q = chunk_seq(p, r.b);
      } while (r.q.n == 0);
    }
  }
  r.length = r.q.s + min((r.j + 1) * per, r.q.n) + p.gap;
}
__device__ __forceinline__ int64_t chunk_share(const ChunkParams& p, int64_t line, int parts) {
  return max((line + parts - 1) / parts, static_cast<int64_t>(p.least));
}

// A pool as {64 columns, slots, column blocks, heads, pages}; one load brings `slots` slots and `blocks` blocks of a page and head.
inline bool encode_pages(CUtensorMap* map, const void* base, int dim, int hkv, int pages, int64_t stride_p, int64_t stride_h, int64_t stride_s,
                         uint32_t slots, uint32_t blocks) {
  const uint64_t dims[5] = {64, PAGE, static_cast<uint64_t>(dim / 64), static_cast<uint64_t>(hkv), static_cast<uint64_t>(pages)};
  const uint64_t strides[4] = {static_cast<uint64_t>(stride_s) * 2, 128, static_cast<uint64_t>(stride_h) * 2, static_cast<uint64_t>(stride_p) * 2};
  const uint32_t box[5] = {64, slots, blocks, 1, 1};
  return encode_map_bf16_sw128(map, base, 5, dims, strides, box);
}

// Attention of calls with few tokens per sequence (chunk_few.cu): whether it takes one, its workspace and its launch.
bool chunk_takes_few(int batch, int tokens, int hkv, int group);
int64_t chunk_few_workspace_bytes(int dim);
int launch_chunk_few(ChunkParams p, const b200_chunk_attention_args& a, cudaStream_t stream);

}  // namespace b200
