// New tokens of a packed batch on their way into the paged cache: queries and keys rotated, keys and values written behind what each
// sequence holds.
//   angle[t, i] = position[axis(i)][t] * inv_freq[i],  (a, b) = (x[i], x[i + R/2]) -> (a cos - b sin, b cos + a sin),  i < R/2
// The rotation's position and the place in the cache are two things: the first comes with every token (and axis, for images and
// video), the second is pos[b] + the token's number in its sequence.
// Positions run far: the product position * inv_freq in 32 bits is off by half a unit in its last place, 0.004 radians at 100 000, so
// it is formed in 64 bits, in turns, and only what is left of the last turn goes on in 32 (off by 2^-25 of half a turn).  The pair is
// rotated in 32 bits and rounded once.
// Bound: memory; every row is read and written once.  With 10 heads' rows of 256 to rotate and 2 to copy per token 32 768 tokens take 67.1 us,
// 6.0 TB/s of 6.5, 8300 tokens 19.7 (what a CTA does once, the places and the angles, is a sixth of it), 32 tokens 3.1.  A row in hand and one
// on its way to a thread: four on their way cost 80 registers and 81 us, one at a time with a division per row 69.
#include "b200_attn.h"
#include "common.cuh"

namespace b200 {

constexpr int RA_THREADS = 256;
constexpr int RA_MAX_TOKENS = 8;   // per CTA
constexpr int RA_RESIDENT = 6;     // CTAs on an SM

struct RopeAppendParams {
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16 *q_out, *k_cache, *v_cache;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h, o_t, kc_p, kc_h, kc_s, vc_p, vc_h, vc_s, bt_b, pid_a;
  const int32_t *block_table, *cu_seqlens, *freq_axis;
  const int64_t* pos;
  const void* position_ids;
  const float* inv_freq;
  int ids_are_int64, axes, batch, tokens, num_pages, max_pages, hq, hkv, dim, rot_half, per_cta;
};

// The sequence that packed row t belongs to, -1 where none does; the whole warp, 32 candidates at a time.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int batch, int t, int lane) {
  int lo = 0, n = batch + 1;  // the largest b in [lo, lo + n) with cu[b] <= t
  while (n > 1) {
    const int step = (n + 31) / 32, i = lo + lane * step;
    const int below = __popc(__ballot_sync(0xffffffffu, lane * step < n && cu[i] <= t));
    if (below == 0) return -1;
    n = min(step, n - (below - 1) * step);
    lo += (below - 1) * step;
  }
  return lo < batch ? lo : -1;
}

__global__ void __launch_bounds__(RA_THREADS)
rope_append_kernel(const __grid_constant__ RopeAppendParams p) {
  extern __shared__ __align__(16) float2 turn[];  // [tokens of the CTA][R/2] sine, cosine
  __shared__ int64_t page_of[RA_MAX_TOKENS];     // -1: no place in the cache, -2: no sequence
  __shared__ int slot_of[RA_MAX_TOKENS];
  pdl_chain();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int t0 = blockIdx.x * p.per_cta, count = min(p.per_cta, p.tokens - t0);
  // A thread's units of two vectors of 8, rotated ones with their partners, the others in neighbours: the same of every row (token and head)
  // that it takes.  The next row is asked for before the one in hand goes out, the first before anything else.
  const int units = p.dim / 16, pairs = p.rot_half / 8, rotated = p.hq + p.hkv, heads = rotated + p.hkv, step = RA_THREADS / units;
  const int u = tid % units, first = u < pairs ? u : 2 * u, second = u < pairs ? u + pairs : 2 * u + 1;
  int n = tid / units / heads, h = tid / units - n * heads;
  if (tid >= step * units) n = count;            // threads that are left over
  auto load = [&](uint4& a, uint4& b) {
    const int64_t t = t0 + n;
    const __nv_bfloat16* src = h < p.hq ? p.q + t * p.q_t + h * p.q_h
                                        : h < rotated ? p.k + t * p.k_t + (h - p.hq) * p.k_h : p.v + t * p.v_t + (h - rotated) * p.v_h;
    a = reinterpret_cast<const uint4*>(src)[first];
    b = reinterpret_cast<const uint4*>(src)[second];
  };
  uint4 next_a, next_b;
  if (n < count) load(next_a, next_b);
  for (int i = tid; i < count * p.rot_half; i += RA_THREADS) {
    const int token = i / p.rot_half, f = i - token * p.rot_half;
    const int axis = p.axes > 1 ? min(max(p.freq_axis[f], 0), p.axes - 1) : 0;
    const int64_t at = axis * p.pid_a + t0 + token;
    const double id = p.ids_are_int64 ? static_cast<double>(static_cast<const int64_t*>(p.position_ids)[at])
                                      : static_cast<double>(static_cast<const int32_t*>(p.position_ids)[at]);
    const double turns = id * static_cast<double>(p.inv_freq[f]) * 0.15915494309189533577;  // 1 / (2 pi)
    float2 sc;
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &sc.x, &sc.y);
    turn[i] = sc;
  }
  for (int i = warp; i < count; i += RA_THREADS / 32) {
    const int t = t0 + i, b = sequence_of(p.cu_seqlens, p.batch, t, lane);
    if (lane == 0) {
      int64_t page = -2;
      const int begins = b >= 0 ? p.cu_seqlens[b] : 0;
      if (b >= 0 && begins <= t) {  // (else cu_seqlens does not ascend, and the place would be a held token's)
        const int64_t at = p.pos[b] + t - begins;
        page = -1;
        if (at >= 0 && at / PAGE < p.max_pages) page = p.block_table[b * p.bt_b + at / PAGE];
        if (page < 0 || page >= p.num_pages) page = -1;
        slot_of[i] = static_cast<int>(at & (PAGE - 1));
      }
      page_of[i] = page;
    }
  }
  __syncthreads();
  while (n < count) {
    uint4 a = next_a, b = next_b;
    const int token = n, head = h;
    for (h += step; h >= heads; h -= heads) ++n;
    if (n < count) load(next_a, next_b);
    const int64_t t = t0 + token, page = page_of[token];
    if (head < p.hq ? page == -2 : page < 0) continue;
    __nv_bfloat16* dst = head < p.hq   ? p.q_out + t * p.o_t + head * p.dim
                         : head < rotated ? p.k_cache + page * p.kc_p + (head - p.hq) * p.kc_h + slot_of[token] * p.kc_s
                                          : p.v_cache + page * p.vc_p + (head - rotated) * p.vc_h + slot_of[token] * p.vc_s;
    if (u < pairs && head < rotated) {
      uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
      const float4* angles = reinterpret_cast<const float4*>(turn + token * p.rot_half + u * 8);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float4 sc = angles[e];             // sine, cosine of two angles
        float f0, g0, f1, g1;
        rope_pair(bf16_lo(wa[e]), bf16_lo(wb[e]), sc.x, sc.y, f0, g0);
        rope_pair(bf16_hi(wa[e]), bf16_hi(wb[e]), sc.z, sc.w, f1, g1);
        wa[e] = pack_bf16(f0, f1);
        wb[e] = pack_bf16(g0, g1);
      }
      a = make_uint4(wa[0], wa[1], wa[2], wa[3]);
      b = make_uint4(wb[0], wb[1], wb[2], wb[3]);
    }
    reinterpret_cast<uint4*>(dst)[first] = a;
    reinterpret_cast<uint4*>(dst)[second] = b;
  }
}

static bool mult8(int64_t x) { return (x & 7) == 0; }

}  // namespace b200

using namespace b200;

extern "C" int b200_paged_kv_append_rope(const b200_rope_append_args* args, b200_stream_t stream) {
  const b200_rope_append_args& a = *args;
  constexpr int64_t most = 0x7fffffff;
  B200_REQUIRE(a.batch > 0 && a.batch < most && a.total_tokens >= 0 && a.total_tokens <= most && a.num_pages > 0 && a.num_pages <= most &&
                   a.max_pages > 0 && a.max_pages <= most,
               "paged_kv_append_rope: empty shape, or more than 2^31 of something");
  B200_REQUIRE(a.num_q_heads > 0 && a.num_kv_heads > 0 && a.num_q_heads <= 1024 && a.num_kv_heads <= 1024,
               "paged_kv_append_rope: heads must be in [1, 1024] (got %lld/%lld)", static_cast<long long>(a.num_q_heads),
               static_cast<long long>(a.num_kv_heads));
  B200_REQUIRE(a.head_dim >= 16 && a.head_dim <= 512 && a.head_dim % 16 == 0,
               "paged_kv_append_rope: head_dim must be a multiple of 16 up to 512 (got %lld)", static_cast<long long>(a.head_dim));
  B200_REQUIRE(a.rotary_dim >= 16 && a.rotary_dim <= a.head_dim && a.rotary_dim % 16 == 0,
               "paged_kv_append_rope: rotary_dim must be a multiple of 16 up to head_dim (got %lld)", static_cast<long long>(a.rotary_dim));
  B200_REQUIRE(a.axes >= 1 && a.axes <= most && (a.axes == 1 || a.freq_axis != nullptr), "paged_kv_append_rope: several axes need freq_axis");
  B200_REQUIRE(aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.q_out) && aligned16(a.k_cache) && aligned16(a.v_cache) &&
                   mult8(a.q_stride_t) && mult8(a.q_stride_h) && mult8(a.k_stride_t) && mult8(a.k_stride_h) && mult8(a.v_stride_t) &&
                   mult8(a.v_stride_h) && mult8(a.out_stride_t) && mult8(a.kc_stride_p) && mult8(a.kc_stride_h) && mult8(a.kc_stride_s) &&
                   mult8(a.vc_stride_p) && mult8(a.vc_stride_h) && mult8(a.vc_stride_s),
               "paged_kv_append_rope: tensors must be 16-byte aligned with strides that are multiples of 8");
  if (a.total_tokens == 0) return OK;
  RopeAppendParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(a.q), p.k = static_cast<const __nv_bfloat16*>(a.k), p.v = static_cast<const __nv_bfloat16*>(a.v);
  p.q_out = static_cast<__nv_bfloat16*>(a.q_out);
  p.k_cache = static_cast<__nv_bfloat16*>(a.k_cache), p.v_cache = static_cast<__nv_bfloat16*>(a.v_cache);
  p.q_t = a.q_stride_t, p.q_h = a.q_stride_h, p.k_t = a.k_stride_t, p.k_h = a.k_stride_h, p.v_t = a.v_stride_t, p.v_h = a.v_stride_h;
  p.o_t = a.out_stride_t;
  p.kc_p = a.kc_stride_p, p.kc_h = a.kc_stride_h, p.kc_s = a.kc_stride_s;
  p.vc_p = a.vc_stride_p, p.vc_h = a.vc_stride_h, p.vc_s = a.vc_stride_s;
  p.bt_b = a.bt_stride_b, p.pid_a = a.ids_stride_a;
  p.block_table = a.block_table, p.cu_seqlens = a.cu_seqlens, p.freq_axis = a.freq_axis, p.pos = a.pos;
  p.position_ids = a.position_ids, p.inv_freq = a.inv_freq;
  p.ids_are_int64 = a.ids_are_int64 != 0, p.axes = a.axes, p.batch = a.batch, p.tokens = a.total_tokens;
  p.num_pages = a.num_pages, p.max_pages = a.max_pages;
  p.hq = a.num_q_heads, p.hkv = a.num_kv_heads, p.dim = a.head_dim, p.rot_half = a.rotary_dim / 2;
  // a CTA per token until the device is full, then as many tokens to a CTA as make whole waves of it
  const int64_t room = static_cast<int64_t>(RA_RESIDENT) * sm_count(), waves = (a.total_tokens + room * RA_MAX_TOKENS - 1) / (room * RA_MAX_TOKENS);
  p.per_cta = static_cast<int>((a.total_tokens + room * waves - 1) / (room * waves));
  const int smem = p.per_cta * p.rot_half * static_cast<int>(sizeof(float2));  // 16 KB at most
  launch_pdl(chain_overlap(), rope_append_kernel, dim3((p.tokens + p.per_cta - 1) / p.per_cta), dim3(RA_THREADS), smem,
             reinterpret_cast<cudaStream_t>(stream), p);
  return check_launch("paged_kv_append_rope");
}
