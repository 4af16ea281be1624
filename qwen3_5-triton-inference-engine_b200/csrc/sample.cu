// The next token of every row of logits, from one given uniform number per row.
//   order: larger logit first, equal ones by index.  Kept is the shortest of the prefixes that top_k, min_p and top_p name:
//     top_k    its first top_k tokens
//     min_p    those with w >= min_p,  w = exp((x - max) / temperature)
//     top_p    the fewest whose weights reach top_p of the sum over what the other two kept
//   id = the first kept token, by index, at which the running sum of kept weights exceeds uniform times the whole.
//
// A row belongs to a cluster of CTAs, which hold it in shared memory or, where more rows then run at once, read it again from the L2: it comes
// from HBM once.  No sorting: a histogram by the distance from the largest, counts for top_k and weights for top_p, summed over the cluster
// through distributed shared memory, names the bin in which the border of a prefix lies; the logits of that bin go to every CTA as a list and are
// compared with one another.  A bin with too many for the list (many equal ones) is searched by the digits of the logit's bits, 11, 11 and 10 of
// them.  Where min_p or top_k leave few tokens, these go to one CTA and are finished there, after one more walk.  Else every warp sums the kept
// weights of its stretch of the row, which for the bins above the border's the walk that makes the list does on its way, and the warp in whose
// stretch the wanted sum lies walks through it.
//
// Which token a number falls on is decided by long sums (up to 2^18 weights of which each may be 2^-18 of the whole), so a sum in 32 bits
// picks a neighbour now and then.  Weights are whole numbers of units of 2^-44 of the largest: their sums are exact, in any order, and equal
// calls give equal ids.  A weight is right to about 2^-28 of itself, and then cut to whole units (half a unit low on the average), so that a sum of n of
// them may be n units low, 2^-25 of the largest for 2^19 tokens that weigh next to nothing:
//   t = x c + (3 * 2^13 - max c), c = log2(e) / temperature, in 64 bits: its lowest 38 bits are the fraction of the exponent to base 2, of which
//   six name an entry of a table of 2^(j/64), and 23 more go on as r < 1/64 to a polynomial of degree 3 for 2^r in 32-bit floats.
// The errors of 2^-28 mostly cancel over many different logits, but for 2^-30 that the fraction's cut makes all of them low.
// The bins are 64ths of a factor of two, the upper half of t as it stands.
//
// Bound by instructions: without a top_k two walks weigh every token after the one that finds the largest, together 109 instructions a token and
// up to two additions in shared memory.  256 rows of 248 320 floats, top_p 0.95: 389 us, 39 at the memory's rate; without the additions
// it were 80 us less; rows so flat that most tokens share a few bins 931.  Few rows wait for their CTAs: seven meetings of the cluster (five with a
// small top_k, three without filters), between them the bins cleared, exchanged and summed, make 22 us of one row of 248 320, 12 without filters.
#include "b200_attn.h"
#include "common.cuh"

#include <cmath>

namespace b200 {

constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32;
constexpr int SA_MAX_CLUSTER = 16;
constexpr int SA_MAX_SLICE = 32768;       // tokens that a CTA holds
constexpr uint32_t SA_BINS = 2048;
constexpr int SA_AHEAD = 4;               // loads of a thread on their way
constexpr int SA_LIST = 1024;             // most candidates of a border that are compared with one another
constexpr int SA_SHORT = 256;             // largest top_k that is looked for among the threads' largest (half of one CTA's threads)
constexpr int SA_UNIT = 44;               // the largest weight is 2^44
constexpr int SA_MAX_N = 1 << 19;         // the sum of all is below 2^63, the upper halves' below 2^32

struct SampleParams {
  const void* logits;
  int64_t row_stride;
  int rows, n;
  const float *uniform, *temperature, *top_p, *min_p;  // NULL: the value for all rows
  const int32_t* top_k;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int64_t* ids;
  int per_warp;                           // vectors of a warp's stretch
  uint32_t table[64];                     // 2^(30 + j/64)
  float poly[4];                          // 2^23 + 2^29 (2^r - 1) in powers of v - 1.5, r = (v - 1) / 64
};

// larger float, larger key, one key for both zeros; NaN never comes here
__device__ __forceinline__ uint32_t float_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_float(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

struct RowWeights {
  double c, offset;
  const uint32_t* table;
  float a0, a1, a2, a3;
  __device__ __forceinline__ double exponent(float x) const { return fma(static_cast<double>(x), c, offset); }
  // 64ths of a factor of two below the largest, rounded up; what is far below leaves the binade of 3 * 2^13 and gets some large number
  __device__ __forceinline__ static uint32_t below(double t) { return 0x40d80000u - static_cast<uint32_t>(__double2hiint(t)); }
  // Bins, highest first: 64 to a factor of two over the first 16 factors, where borders lie, 32 over 32 more, behind which nothing weighs anything
  __device__ __forceinline__ uint32_t bin(float x) const {
    const uint32_t k = below(exponent(x));
    return min(min(k, (k >> 1) + 512), SA_BINS);
  }
  // weight of a logit up to the largest
  __device__ __forceinline__ uint64_t operator()(float x) const {
    const double t = exponent(x);
    const uint32_t lo = static_cast<uint32_t>(__double2loint(t));
    const float d = __uint_as_float((lo >> 9) | 0x3f800000u) - 1.5f;
    const float y = fmaf(fmaf(fmaf(a3, d, a2), d, a1), d, a0);
    const uint32_t e = table[__double2hiint(t) & 63];
    const uint32_t m = e + __umulhi(e, __float_as_uint(y) << 3 & 0x3fffff8u);  // 2^30 to 2^31
    uint64_t w = static_cast<uint64_t>(m) << (SA_UNIT - 30);
    asm("shr.b64 %0, %0, %1;" : "+l"(w) : "r"((below(t) + 63) >> 6));  // (64 and more: nothing is left)
    return w;
  }
};

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct alignas(16) SampleShared {
  union {
    uint32_t hist[2][SA_BINS];            // counts, or weights' lower and upper halves
    struct {                              // once the bins have been summed up
      float cand[SA_LIST];                // every CTA's candidates, SA_LIST / cluster places each
      uint32_t cand_id[SA_LIST];
      float list[SA_LIST];                // the same without gaps
      uint32_t list_id[SA_LIST];
      uint64_t list_w[SA_LIST];
    };
  };
  uint64_t total[SA_BINS];                // of the whole row
  uint32_t table[64];
  float warp_max[SA_WARPS];
  uint32_t cta_max[SA_MAX_CLUSTER];
  uint64_t warp_sum[SA_WARPS], cta_sum[SA_MAX_CLUSTER];
  uint32_t warp_equal[SA_WARPS];
  uint64_t cta_equal[SA_MAX_CLUSTER];
  uint32_t cand_count[SA_MAX_CLUSTER];
  uint64_t scan[SA_WARPS];
  uint64_t found_above;
  int found_bin;
  uint32_t found_logit;                   // its bits
  uint32_t fill;
};

// RESIDENT: the cluster holds the row in shared memory; else it reads it again, from the L2.
template <typename T, bool RESIDENT>
__global__ void __launch_bounds__(SA_THREADS, 2)
sample_kernel(const __grid_constant__ SampleParams p) {
  constexpr int V = 16 / sizeof(T);       // tokens of a 16-byte vector
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SampleShared& sm = *reinterpret_cast<SampleShared*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t csize;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));
  const uint32_t rank = cluster_ctarank();
  const int row = blockIdx.x / csize;
  // the row as aligned vectors, of which the first and last may stand out of it
  const T* x_row = static_cast<const T*>(p.logits) + row * p.row_stride;
  const int out = static_cast<int>((reinterpret_cast<uintptr_t>(x_row) & 15) / sizeof(T));
  const int vectors = (out + p.n + V - 1) / V;
  const int v0 = (rank * SA_WARPS + warp) * p.per_warp, count = max(0, min(p.per_warp, vectors - v0));  // this warp's
  const int first = v0 * V - out, quads = count * (V / 4);  // its first token, four tokens at a time
  float* mine = reinterpret_cast<float*>(smem_raw + sizeof(SampleShared)) + warp * p.per_warp * V;
  cluster_started();
  if (tid < 64) sm.table[tid] = p.table[tid];
  const float temperature = p.temperature ? p.temperature[row] : p.temperature_all;
  const float top_p = p.top_p ? p.top_p[row] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[row] : p.min_p_all;
  const int top_k = p.top_k ? p.top_k[row] : p.top_k_all;
  const double u = fmin(fmax(static_cast<double>(p.uniform[row]), 0.0), 1.0);

  // Four tokens of the row as it stands in memory; -inf for what is not in it or not a number.
  auto fetch = [&](int i, float (&f)[4]) {
    const int at = first + i * 4;
    if (at >= 0 && at + 4 <= p.n) {
      if (V == 4) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(x_row + at));
        f[0] = x.x, f[1] = x.y, f[2] = x.z, f[3] = x.w;
      } else {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(x_row + at));
        f[0] = bf16_lo(x.x), f[1] = bf16_hi(x.x), f[2] = bf16_lo(x.y), f[3] = bf16_hi(x.y);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = at + e >= 0 && at + e < p.n ? static_cast<float>(x_row[at + e]) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = fmaxf(f[e], -INFINITY);
  };

  // ---- the row's maximum
  float own = -INFINITY;                   // of this thread's tokens
#pragma unroll 1
  for (int i0 = lane; i0 < quads; i0 += 32 * SA_AHEAD) {
    float f[SA_AHEAD][4];
#pragma unroll
    for (int k = 0; k < SA_AHEAD; ++k) fetch(min(i0 + k * 32, quads - 1), f[k]);
#pragma unroll
    for (int k = 0; k < SA_AHEAD; ++k) {
      if (i0 + k * 32 < quads) own = fmaxf(own, fmaxf(fmaxf(f[k][0], f[k][1]), fmaxf(f[k][2], f[k][3])));
      if (RESIDENT && i0 + k * 32 < quads) *reinterpret_cast<float4*>(mine + (i0 + k * 32) * 4) = make_float4(f[k][0], f[k][1], f[k][2], f[k][3]);
    }
  }
  // Where nothing but the largest weighs anything, because it is infinite or the next float is 64 factors of two away: it counts as zero, all
  // else as nothing.
  bool alone = false;
  float top = 0.f;
  auto element = [&](int i, float (&f)[4]) {
    if (RESIDENT) {
      const float4 x = *reinterpret_cast<const float4*>(mine + i * 4);
      f[0] = x.x, f[1] = x.y, f[2] = x.z, f[3] = x.w;
    } else {
      fetch(i, f);
    }
    if (alone) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = f[e] == top ? 0.f : -INFINITY;
    }
  };
  // All of the warp's stretch, `visit` called with the number of four tokens and the four; from the L2 a few on their way at a time.
  auto walk = [&](auto visit) {
    constexpr int AHEAD = RESIDENT ? 1 : SA_AHEAD;
#pragma unroll 1
    for (int i0 = lane; i0 < quads; i0 += 32 * AHEAD) {
      float f[AHEAD][4];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) element(min(i0 + k * 32, quads - 1), f[k]);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (AHEAD == 1 || i0 + k * 32 < quads) visit(i0 + k * 32, f[k]);
    }
  };
  float best = warp_max(own);
  if (lane == 0) sm.warp_max[warp] = best;
  __syncthreads();
  cluster_all_started();
  if (tid < csize) {
    float m = sm.warp_max[0];
    for (int i = 1; i < SA_WARPS; ++i) m = fmaxf(m, sm.warp_max[i]);
    peer_store(peer_smem(&sm.cta_max[rank], tid), __float_as_uint(m));
  }
  cluster_sync();
  best = -INFINITY;
  for (int i = 0; i < csize; ++i) best = fmaxf(best, __uint_as_float(sm.cta_max[i]));

  const float temp = fminf(fmaxf(temperature, 1e-6f), 3.402823466e38f);  // (infinity as the largest float: c and the borders below stay finite)
  const bool greedy = !(temperature > 0.f) || best == -INFINITY;
  RowWeights weight;
  weight.table = sm.table;
  weight.a0 = p.poly[0], weight.a1 = p.poly[1], weight.a2 = p.poly[2], weight.a3 = p.poly[3];
  weight.c = 1.4426950408889634 / static_cast<double>(temp);
  if (!greedy && !(fabs(static_cast<double>(best) * weight.c) < 1073741824.0)) alone = true, top = best, best = 0.f, own = own == top ? 0.f : -INFINITY;
  weight.offset = 24576.0 - static_cast<double>(best) * weight.c;

  uint64_t sum = 0;                       // of kept weights of this thread
  int listed = 0;                         // candidates in the list
  // kept: logits above `border`, and the first `ties` of those that equal it
  float border = -INFINITY;
  uint32_t ties = 0;

  // Counts or weights of the logits by the bins that `bin_for` gives them (SA_BINS: none), summed over the cluster, and the bin in which the
  // sum from above reaches `want` (weights, want 0: top_p of everything, found first).  `largest`: of each thread's largest only.  Results in
  // sm.found_*, bin -1: not reached.
  auto search = [&](bool weights, bool largest, uint64_t want, auto bin_for) {
    for (uint32_t i = tid; i < SA_BINS; i += SA_THREADS) {
      sm.hist[0][i] = 0;
      if (weights) sm.hist[1][i] = 0;
    }
    __syncthreads();
    if (largest) {
      const uint32_t bin = bin_for(own);
      if (bin < SA_BINS) atomicAdd(&sm.hist[0][bin], 1u);
    } else if (weights) {
      walk([&](int, const float (&f)[4]) {
        uint32_t bin[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) bin[e] = bin_for(f[e]);
        if (min(min(bin[0], bin[1]), min(bin[2], bin[3])) >= SA_BINS) return;
        uint64_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = weight(f[e]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (bin[e] < SA_BINS) {
            // a 64-bit addition takes three times as long as two of 32 bits, of which small weights mostly need one
            const uint32_t low = static_cast<uint32_t>(w[e]), sum = atomicAdd(&sm.hist[0][bin[e]], low) + low;
            const uint32_t high = static_cast<uint32_t>(w[e] >> 32) + (sum < low);
            if (high) atomicAdd(&sm.hist[1][bin[e]], high);
          }
      });
    } else {
      walk([&](int, const float (&f)[4]) {
        uint32_t bin[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) bin[e] = bin_for(f[e]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (bin[e] < SA_BINS) atomicAdd(&sm.hist[0][bin[e]], 1u);
      });
    }
    cluster_sync();
    // every CTA sums its share of the bins and tells all of them
    const int share = SA_BINS / csize;
    for (int i = tid; i < share; i += SA_THREADS) {
      const int bin = rank * share + i;
      uint64_t sum = 0;
#pragma unroll 8
      for (int c = 0; c < csize; ++c) {
        const uint32_t there = peer_smem(&sm.hist[0][bin], c);
        sum += peer_load(there);
        if (weights) sum += static_cast<uint64_t>(peer_load(there + SA_BINS * 4)) << 32;
      }
#pragma unroll 4
      for (int c = 0; c < csize; ++c) peer_store(peer_smem(&sm.total[bin], c), sum);
    }
    cluster_sync();
    // sums from the first bin on, four bins to a thread
    constexpr int PER = SA_BINS / SA_THREADS;
    uint64_t part[PER], all = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) all += part[i] = sm.total[tid * PER + i];
    uint64_t upto = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    if (lane == 31) sm.scan[warp] = upto;
    __syncthreads();
    uint64_t whole = 0, above = upto - all;
    for (int i = 0; i < SA_WARPS; ++i) {
      if (i < warp) above += sm.scan[i];
      whole += sm.scan[i];
    }
    if (weights && want == 0) {
      const uint64_t z = whole + (ties ? ties * weight(border) : 0);
      want = static_cast<uint64_t>(ceil(fmax(static_cast<double>(top_p), 0.0) * static_cast<double>(z)));
      want = want == 0 ? 1 : min(want, z);
    }
    if (whole < want) {                    // not reached
      if (tid == 0) sm.found_bin = -1, sm.found_above = whole;
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (above < want && above + part[i] >= want) sm.found_bin = tid * PER + i, sm.found_above = above;
        above += part[i];
      }
    }
    __syncthreads();
    return want;
  };
  // Every logit that `want` takes, with its index, into the lists of the CTAs in [0, to).  Their number; -1 if some CTA has more than its places.
  // `other` sees the rest.
  auto gather = [&](int to, auto want, auto other) {
    const int places = SA_LIST / csize;
    if (tid == 0) sm.fill = 0;
    __syncthreads();
    walk([&](int i, const float (&f)[4]) {
      bool some[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) some[e] = want(f[e]);
      other(f);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (some[e]) {
          const uint32_t at = atomicAdd(&sm.fill, 1u);
          if (at < places) sm.list[at] = f[e], sm.list_id[at] = first + i * 4 + e;
        }
    });
    __syncthreads();
    const int have = min(sm.fill, static_cast<uint32_t>(places));
    for (int i = tid; i < have * to; i += SA_THREADS) {
      const int c = i / have, n = i - c * have;
      peer_store(peer_smem(&sm.cand[rank * places + n], c), __float_as_uint(sm.list[n]));
      peer_store(peer_smem(&sm.cand_id[rank * places + n], c), sm.list_id[n]);
    }
    if (tid < csize) peer_store(peer_smem(&sm.cand_count[rank], tid), sm.fill);
    cluster_sync();
    int n = 0;
    bool fits = true;
    for (int c = 0; c < csize; ++c) {
      const int there = min(sm.cand_count[c], static_cast<uint32_t>(places));
      fits &= sm.cand_count[c] <= places;
      for (int i = tid; i < there; i += SA_THREADS) {
        const float f = sm.cand[c * places + i];
        sm.list[n + i] = f;
        sm.list_id[n + i] = sm.cand_id[c * places + i];
        sm.list_w[n + i] = weight(f);
      }
      n += there;
    }
    __syncthreads();
    return fits ? n : -1;
  };
  // Sum over the CTA.
  auto cta_sum = [&](uint64_t v) {
    v = warp_sum64(v);
    __syncthreads();
    if (lane == 0) sm.scan[warp] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < SA_WARPS; ++i) v += sm.scan[i];
    return v;
  };
  // The rest of a row of which the list holds what min_p keeps of the first top_k, and some more; every entry is compared with all others.
  auto finish = [&](int n, uint32_t top_k) {
    const bool there = tid < n;
    const float f = there ? sm.list[tid] : 0.f;
    const uint32_t id = there ? sm.list_id[tid] : 0;
    uint64_t w = there ? sm.list_w[tid] : 0, before = 0;
    uint32_t place = 0;
    for (int j = 0; j < n; ++j) {
      const float g = sm.list[j];
      if (g > f || (g == f && sm.list_id[j] < id)) ++place, before += sm.list_w[j];
    }
    if (place >= top_k) w = 0;
    const uint64_t z = cta_sum(w);
    if (top_p < 1.f && static_cast<double>(before) >= fmax(static_cast<double>(top_p), 0.0) * static_cast<double>(z) && place > 0) w = 0;
    const uint64_t whole = cta_sum(w);
    if (there) sm.list_w[tid] = w;
    __syncthreads();
    const uint64_t target = min(static_cast<uint64_t>(u * static_cast<double>(whole)), whole - 1);
    uint64_t sum = 0;
    for (int j = 0; j < n; ++j)
      if (sm.list_id[j] < id) sum += sm.list_w[j];
    if (there && sum <= target && target < sum + w) p.ids[row] = id;
  };
  // The logit at which the sum over those above `border` reaches `want`, and how much of it is left for those equal to it.
  enum { NOT_REACHED, FOUND, BY_DIGITS };
  auto select = [&](bool weights, uint64_t want, float& at, uint64_t& rest) {
    // the bin, then its logits compared with one another
    want = search(weights, false, want, [&](float f) { return f > border ? weight.bin(f) : SA_BINS; });
    const int bin = sm.found_bin;
    rest = want - sm.found_above;
    if (bin < 0) return NOT_REACHED;
    sum = 0;
    const int n = gather(csize, [&](float f) { return weight.bin(f) == bin && f > border; }, [&](const float (&f)[4]) {
      // on the way, what lies above the bin is summed up for the draw
      bool some[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) some[e] = weight.bin(f[e]) < bin && f[e] > border;
      if (!weights || !(some[0] | some[1] | some[2] | some[3])) return;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t w = weight(f[e]);
        sum += some[e] ? w : 0;
      }
    });
    listed = n;
    if (n >= 0) {
      // every CTA compares its share of the candidates with all of them, and the one that has the border's tells the others
      for (int i = tid * csize + rank; i < n; i += SA_THREADS * csize) {
        const float f = sm.list[i];
        uint64_t above = 0, here = 0;
        for (int j = 0; j < n; ++j) {
          const uint64_t amount = weights ? sm.list_w[j] : 1;
          if (sm.list[j] > f) above += amount;
          else if (sm.list[j] == f) here += amount;
        }
        if (above < rest && above + here >= rest) {  // equal ones say the same
          for (int c = 0; c < csize; ++c) {
            peer_store(peer_smem(&sm.found_logit, c), __float_as_uint(f));
            peer_store(peer_smem(&sm.found_above, c), above);
          }
        }
      }
      cluster_sync();
      at = __uint_as_float(sm.found_logit);
      rest -= sm.found_above;
      return FOUND;
    }
    // too many of them: digit by digit
    uint32_t prefix = 0;
    rest = want;
    const int shifts[3] = {21, 10, 0};
#pragma unroll 1
    for (int d = 0; d < 3; ++d) {
      const int bits = d < 2 ? 11 : 10, shift = shifts[d];
      const uint32_t last = (1u << bits) - 1;
      search(weights, false, rest, [&](float f) {
        const uint32_t k = float_key(f);
        const bool some = f > border && (d == 0 || k >> (shift + bits) == prefix) && weight.bin(f) < SA_BINS;
        return some ? last - ((k >> shift) & last) : SA_BINS;
      });
      prefix = prefix << bits | (last - sm.found_bin);
      rest -= sm.found_above;
      __syncthreads();
    }
    at = key_float(prefix);
    return BY_DIGITS;
  };

  if (greedy) {
    // the lowest index of the largest: each warp's, each CTA's, the cluster's
    uint32_t low = 0xffffffffu;
    walk([&](int i, const float (&f)[4]) {
#pragma unroll
      for (int e = 3; e >= 0; --e) {
        const int at = first + i * 4 + e;
        if (f[e] == best && at >= 0) low = min(low, static_cast<uint32_t>(at));
      }
    });
    low = __reduce_min_sync(0xffffffffu, low);
    if (lane == 0) sm.warp_equal[warp] = low;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < SA_WARPS; ++i) low = min(low, sm.warp_equal[i]);
      peer_store(peer_smem(&sm.cta_equal[rank], 0), static_cast<uint64_t>(low));
    }
    cluster_sync();
    if (rank == 0 && tid == 0) {
      for (int i = 0; i < csize; ++i) low = min(low, static_cast<uint32_t>(sm.cta_equal[i]));
      p.ids[row] = low;
    }
    return;
  }

  float least = -INFINITY;                 // the least logit whose weight is not below min_p
  if (min_p > 0.f) {
    least = best;
    if (min_p < 1.f) {
      const double t = static_cast<double>(best) + static_cast<double>(temp) * log(static_cast<double>(min_p));
      least = static_cast<float>(t);
      if (static_cast<double>(least) < t) least = nextafterf(least, INFINITY);
      least = fminf(least, best);
    }
    border = nextafterf(least, -INFINITY);
  }
  // of those that min_p keeps, so that fewer than top_k may be there, or weigh anything
  // Few tokens are picked out at once and finished as a list: what lies in or above the bin in which the threads' largest reach top_k holds the
  // first top_k and little else, and min_p mostly keeps little.  (32 rows of 248 320, top_k 25 to 50, min_p 0.03 to 0.05: 25 us, by a
  // histogram of all tokens 51.  A min_p that keeps more than the lists hold has walked for nothing: 256 rows under min_p 1e-6 308 us, 188 without.)
  int bin = -1;
  if (top_k > 0 && top_k <= SA_SHORT) {
    search(false, true, top_k, [&](float f) { return f > border ? weight.bin(f) : SA_BINS; });
    bin = sm.found_bin;
  }
  if (bin >= 0 || min_p > 0.f) {
    // a logit that lies below everything in the bin: most are told by a comparison
    const int steps = bin < 1024 ? bin + 1 : 2 * (bin - 512) + 2, most = bin < 0 ? SA_BINS : bin;
    const float far = bin < 0 ? border : __double2float_rd(static_cast<double>(best) - (steps + 1) * 0.015625 / weight.c);
    const int n = gather(1, [&](float f) { return f >= far && f > border && weight.bin(f) <= most; }, [](const float (&)[4]) {});
    if (n >= 0 && n <= SA_THREADS) {
      if (rank == 0) finish(n, top_k > 0 ? top_k : n);
      return;
    }
  }
  if (top_k > 0 && top_k < p.n) {
    float at;
    uint64_t rest;
    const auto how = select(false, top_k, at, rest);
    if (how != NOT_REACHED) border = at, ties = static_cast<uint32_t>(rest);
  }
  bool summed = false;
  if (top_p < 1.f) {
    float at;
    uint64_t rest;
    const auto how = select(true, 0, at, rest);
    const bool inside = how != NOT_REACHED;
    summed = how == FOUND;
    if (inside) border = at;
    const uint64_t w = weight(border);
    const uint64_t need = w == 0 ? ties : (rest + w - 1) / w;
    if (inside || need < ties) ties = static_cast<uint32_t>(need);
  }

  // ---- the draw: kept weights and ties of every warp's stretch
  uint32_t equal = 0;
  if (!summed) {
    sum = 0;
    walk([&](int, const float (&f)[4]) {
      bool some[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        some[e] = f[e] > border;
        equal += f[e] == border;
      }
      if (!(some[0] | some[1] | some[2] | some[3])) return;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t w = weight(f[e]);
        sum += some[e] ? w : 0;
      }
    });
  }
  sum = warp_sum64(sum);
  equal = __reduce_add_sync(0xffffffffu, equal);
  if (lane == 0) sm.warp_sum[warp] = sum, sm.warp_equal[warp] = equal;
  __syncthreads();
  if (summed) {                            // the border's bin, of which the candidates are all
    for (int i = tid; i < listed; i += SA_THREADS) {
      const float f = sm.list[i];
      const int of = (static_cast<int>(sm.list_id[i]) + out) / V / p.per_warp - static_cast<int>(rank) * SA_WARPS;
      if (of < 0 || of >= SA_WARPS) continue;
      if (f > border) atomicAdd(reinterpret_cast<unsigned long long*>(&sm.warp_sum[of]), static_cast<unsigned long long>(sm.list_w[i]));
      else if (f == border) atomicAdd(&sm.warp_equal[of], 1u);
    }
    __syncthreads();
  }
  if (tid < csize) {
    uint64_t s = 0, q = 0;
    for (int i = 0; i < SA_WARPS; ++i) s += sm.warp_sum[i], q += sm.warp_equal[i];
    peer_store(peer_smem(&sm.cta_sum[rank], tid), s);
    peer_store(peer_smem(&sm.cta_equal[rank], tid), q);
  }
  cluster_sync();                          // from here on a CTA reads its own shared memory only
  const uint64_t w_border = ties ? weight(border) : 0;
  uint64_t before = 0, seen = 0, whole = 0, equals = 0;  // of the CTAs in front, of all
  for (int i = 0; i < csize; ++i) {
    if (i == rank) before = whole, seen = equals;
    whole += sm.cta_sum[i];
    equals += sm.cta_equal[i];
  }
  whole += min(equals, static_cast<uint64_t>(ties)) * w_border;
  const uint64_t target = min(static_cast<uint64_t>(u * static_cast<double>(whole)), whole - 1);  // the running sum has to exceed it
  for (int i = 0; i < warp; ++i) before += sm.warp_sum[i], seen += sm.warp_equal[i];
  auto kept_ties = [&](uint64_t s) { return min(s, static_cast<uint64_t>(ties)); };
  const uint64_t start = before + kept_ties(seen) * w_border;
  const uint64_t end = before + sm.warp_sum[warp] + kept_ties(seen + sm.warp_equal[warp]) * w_border;
  if (target < start || target >= end) return;
  uint64_t running = start;                // the whole warp is in here
  for (int i0 = 0; i0 < quads; i0 += 32) {
    const int i = i0 + lane;
    uint64_t w[4] = {0, 0, 0, 0};
    uint32_t tie[4] = {0, 0, 0, 0};
    if (i < quads) {
      float f[4];
      element(i, f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (f[e] > border) w[e] = weight(f[e]);
        else tie[e] = f[e] == border;
      }
    }
    uint32_t tied = tie[0] + tie[1] + tie[2] + tie[3], upto = tied;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    uint64_t rank_of = seen + upto - tied;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (tie[e] && rank_of++ < ties) w[e] = w_border;
    }
    const uint64_t own = w[0] + w[1] + w[2] + w[3];
    uint64_t sums = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(0xffffffffu, sums, o);
      if (lane >= o) sums += up;
    }
    uint64_t at = running + sums - own;
    if (at <= target && target < at + own) {
      int e = 0;
      while (e < 3 && target >= at + w[e]) at += w[e++];
      p.ids[row] = first + i * 4 + e;
    }
    running += __shfl_sync(0xffffffffu, sums, 31);
    seen += __shfl_sync(0xffffffffu, upto, 31);
    if (running > target) return;
  }
}

// How a call runs: CTAs of a row, and whether they hold it.  The largest clusters of which all rows' fit the device at once, but not less than
// 2000 tokens to a CTA nor more than 65 536; twice as many CTAs where that leaves more than 20 000 to one and two on an SM are enough for all.
// Held is a row of which two shares fit an SM, or of which one does if all CTAs run at once; else it is read again from the L2.  us, top_p 0.9: 1 row
// of 248 320 on 16 CTAs 24.7 (read again 28), 8 34, 4 65; 8 rows on 16 36, 8 44; 32 rows on 8, read again, 67 (held 91), 16 85, 4 86; 256 rows
// on 4, read again, 376, 8 440 (held 581), 16 583; 32 of 65 000 on 4 26 (read again 30), 8 24, 2 39; 128 of 16 000 on 1, 2, 4 24.4 (read
// again 27.7), 22.1, 32.3.
struct SamplePlan {
  int cluster;
  bool resident;
};
static SamplePlan sample_plan(int rows, int n) {
  const int sms = sm_count();
  auto fits = [&](int c) { return c <= 2 ? sms / c : (c == 4 ? sms * 33 : c == 8 ? sms * 15 : sms * 7) / 148; };  // clusters at once
  int c = 1;
  while (c < SA_MAX_CLUSTER && n >= 2 * c * 2000 && rows <= fits(2 * c)) c *= 2;
  while (n > c * 65536) c *= 2;
  if (c < SA_MAX_CLUSTER && n > c * 20000 && rows * c * 2 <= sms * 264 / 148) c *= 2;
  return {c, n <= c * 17000 || (n <= c * SA_MAX_SLICE && rows * c <= sms)};
}

template <typename T>
static int launch_sample(SampleParams& p, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const SamplePlan plan = sample_plan(p.rows, p.n);
  const int vectors = (p.n + 2 * V - 2) / V;  // with the worst alignment
  p.per_warp = (vectors + plan.cluster * SA_WARPS - 1) / (plan.cluster * SA_WARPS);
  int smem = static_cast<int>(sizeof(SampleShared));
  if (plan.resident) smem += p.per_warp * SA_WARPS * 16 * (4 / static_cast<int>(sizeof(T)));
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    constexpr int most = static_cast<int>(sizeof(SampleShared)) + (SA_MAX_SLICE + 64 * SA_WARPS) * 4;
    for (const auto k : {sample_kernel<T, true>, sample_kernel<T, false>})
      if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess ||
          cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
        return fail(ERR_RUNTIME, "sample_rows: cannot raise dynamic shared memory to %d", most);
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  if (launch_pdl_cluster(false, plan.cluster, plan.resident ? sample_kernel<T, true> : sample_kernel<T, false>, dim3(p.rows * plan.cluster),
                         dim3(SA_THREADS), smem, stream, p) != cudaSuccess)
    return fail(ERR_LAUNCH, "sample_rows: %s", cudaGetErrorString(cudaGetLastError()));
  return check_launch("sample_rows");
}

}  // namespace b200

using namespace b200;

extern "C" int b200_sample_rows(const b200_sample_args* args, b200_stream_t stream) {
  const b200_sample_args& a = *args;
  B200_REQUIRE(a.rows >= 0 && a.rows <= 65535 && a.n > 0 && a.n <= SA_MAX_N,
               "sample_rows: needs at most 65535 rows of 1 to %d logits (got %lld, %lld)", SA_MAX_N, static_cast<long long>(a.rows),
               static_cast<long long>(a.n));
  if (a.rows == 0) return OK;
  SampleParams p = {};
  p.logits = a.logits, p.row_stride = a.row_stride, p.rows = a.rows, p.n = a.n;
  p.uniform = a.uniform, p.temperature = a.temperature, p.top_p = a.top_p, p.min_p = a.min_p, p.top_k = a.top_k;
  p.temperature_all = static_cast<float>(a.temperature_all), p.top_p_all = static_cast<float>(a.top_p_all);
  p.min_p_all = static_cast<float>(a.min_p_all);
  p.top_k_all = a.top_k_all >= 1 && a.top_k_all < a.n ? static_cast<int>(a.top_k_all) : 0;
  p.ids = a.ids;
  static const struct Constants {
    uint32_t table[64];
    float poly[4];
    Constants() {
      for (int j = 0; j < 64; ++j) table[j] = static_cast<uint32_t>(std::llrint(std::exp2(30.0 + j / 64.0)));
      // around the middle of the interval, r = 1/128: 2^r = E e^(h (v - 1.5)), E = 2^(1/128), h = ln 2 / 64; what is left out is below 2^-34
      const double E = std::exp2(1.0 / 128), h = std::log(2.0) / 64, one = std::exp2(29.0);
      poly[0] = static_cast<float>(std::exp2(23.0) + (E - 1) * one);
      poly[1] = static_cast<float>(E * h * one);
      poly[2] = static_cast<float>(E * h * h / 2 * one);
      poly[3] = static_cast<float>(E * h * h * h / 6 * one);
    }
  } constants;
  for (int j = 0; j < 64; ++j) p.table[j] = constants.table[j];
  for (int j = 0; j < 4; ++j) p.poly[j] = constants.poly[j];
  const auto st = reinterpret_cast<cudaStream_t>(stream);
  return a.is_bf16 ? launch_sample<__nv_bfloat16>(p, st) : launch_sample<float>(p, st);
}
