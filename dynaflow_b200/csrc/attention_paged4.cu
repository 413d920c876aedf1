// Attention of a step's new tokens over a key/value cache held in pages of 4-bit codes.
//
// A key is s_k n + m_k (16 code values n, one scale s_k and one minimum m_k a token and head), a value likewise:
//   score(key) = scale * (s_k (q . n) + m_k sum(q))
//   out        = (sum p s_v (n_v - 7.5) + sum p (m_v + 7.5 s_v)) / sum p,       p = exp(score - reference)
// so both products run on the codes themselves and the parameters are two multiplications a score.
//
// The codes feed the matrix instructions without a conversion: a 16-bit half with a code in its low four bits
// is, read as fp16, the subnormal number n * 2^-24 (or 16 n * 2^-24 from the next four bits), which the
// matrix units take exactly. Eight codes cost four ANDs and a shift. The powers of two are put back with the
// scores and the result.
//
// The values are counted from the middle of their range because both sums of the result would otherwise grow with the
// number of keys and all but cancel, and the matrix unit cuts its fp32 sums off instead of rounding them (about 2^-23 of
// the sum a step, always towards zero): 65536 keys of N(0, 1) in one warp were 13 % off that way. Codes have no half steps
// (and made into fp16 numbers around zero, one operation a pair, they cost 1.6 us more on 128 requests x 4096 tokens), so
// keys 0-7 of a granule go in as n, keys 8-15 as -(15 - n): the complement of the word, and a weight with the other sign. That
// is level where both halves weigh the same; what they do not is added up by a matrix instruction with rows of ones, and 7.5
// times that is taken off the sums every LEVEL_TILES tiles. Everything is summed in fp32; roundings to fewer bits:
//   * q is scaled by a power of two a row (its largest element to [2^14, 2^15)) and held in fp16: bf16 has 8
//     significant bits, fp16 11, so only elements below 2^-28 of the largest lose any;
//   * p s_v f is held in fp16 for the value product, f a power of two of each column that follows the largest p s_v seen so
//     far and puts it near the upper end of the format: 2^11 when f is chosen, 2^15 at most. A weight is off by 2^-12 of its value
//     (against the 2^-9 of the bf16 result), on codes of at most 7.5; where it is below 2^-25 of the largest, by 2^-36 of the
//     largest. It does not follow s_v alone, nor the largest p: a key with most of the weight may have a value near zero,
//     and a large value next to no weight, and what is left of the other keys is then the result.
//
// Both products are transposed, 16 keys on the rows of m16n8k16 and the query columns (new token x head of the
// group) on its 8 columns:  S^T[16 keys, 8] = K[16, 128] Q^T  and  O^T[128 dims, 8] += V^T[128, 16 keys] P^T.
// A thread's 16 bytes of a key row are four k-steps of A fragments whatever the order of the dimensions, as long
// as Q's fragments use the same order; the value fragments come from transposed 8x8 loads (a 16-bit unit is
// four dimensions of one key, its transposed pair the same four of the next key); P^T from the scores' layout by
// two 8x8 transposes in registers. (A decode step has one query row a head; at 8 columns the work is 1/16 of
// what the tensor pipe would do in the time the bytes take, so it stays on the warp-level instructions: operands
// come from registers, where the codes are unpacked, instead of going through shared or tensor memory again.)
//
// Work: the tiles (32 tokens of a head, two granules) of all requests and heads in one list, cut evenly over the CTAs
// and, inside a CTA, over its warps, whatever the lengths. A warp walks its part on its own: its lanes issue the copies
// of its ring (one contiguous bulk copy a tile, two where a page ends inside it), it keeps its own reference, sums and
// O^T and waits for no other warp. A request and head that lies inside one warp's part is written to the output at
// once; one that is cut between warps is joined in shared memory at the end of the CTA; one that is cut between CTAs
// leaves a partial result each (at most two a CTA), and the CTA that finishes last joins them in the order of the CTAs
// (a counter a cut, which that CTA sets back to zero).
// A request and head costs a warp its queries and its result as well as its tiles, so it counts SEGMENT_COST tiles
// more when the list is cut (without: 16 requests of a few tokens among long ones make one CTA twice as long).
//
// Bound: HBM, 136 bytes a key and head, with the instructions close behind: long caches stream at 5.8 TB/s (the difference
// between 65536 and 32768 tokens, 8 requests, 8 heads: 285 MB in 49 us), where a scheduler issues in about every second cycle. Short
// ones are bound by what lies around that: about 5 us from the lengths over the page table to the first data, 3 to 8 us of
// joins. 128 requests x 4096 tokens, one head: 71 MB in 24.8 us.
// With 9 to 16 columns (4 new tokens of 4 heads, 5 requests of 20000 to 65536 tokens: 244 MB in 82 us) a warp's chain of
// products and softmax is longer than its share of the bytes takes, at two warps a scheduler (246 registers).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "host_util.h"
#include "paged_layout.cuh"
#include "ptx.cuh"

namespace df {
namespace paged {

constexpr int WHERE_PAGED_ATTN = 51;
constexpr float RESCALE_LIMIT = 8.0f;         // the reference moves when a score exceeds it by 2^8
constexpr int WEIGHT_TOP = 11;                // the largest p s_v f when f is chosen: 2^11 at most,
constexpr float WEIGHT_LIMIT = 15.0f;         // and never more than 2^15 (the largest fp16 number is 65504)
constexpr int WEIGHT_SCALE_MAX = 100;         // f is at most 2^100: p f stays in fp32
constexpr int PARTIAL_FLOATS = HEAD_DIM + 4;  // O, reference (log2), sum; padded to 16 bytes
constexpr int REQUESTS_IN_SMEM = 1024;        // requests whose lengths and prefix sums fit into shared memory
constexpr int TILE = 2 * GRANULE;             // tokens
constexpr int TILE_BYTES = 2 * GRANULE_BYTES;
constexpr int LEVEL_TILES = 8;                // tiles between two levellings of the sums (4 new tokens: 81.9 us; 16: 81.6, 4: 82.2, 1: 83.9)
constexpr unsigned SEGMENT_COST = 3;          // tiles (48 requests of 1 to 16384 tokens, 8 heads: 35.0 us; 1: 39.9, 2: 35.1, 4: 35.2)
constexpr unsigned JOIN_COST = 40;            // tiles of 8 columns a CTA does in the time that a join between CTAs takes
constexpr int MAX_COLUMNS = 1 << 20;

struct AttnParams {
  const __nv_bfloat16* q;
  const uint8_t* cache;
  const int* table;
  const int* seq_lens;
  const int* row_starts;  // may be null: request b is row b
  const int* new_lens;    // may be null: one row a request
  __nv_bfloat16* out;
  float* partial;         // [ctas][2][columns][PARTIAL_FLOATS]: what CTAs leave
  float* heads;           // [ctas][warps][columns][PARTIAL_FLOATS]: what warps leave before their end
  int* arrived;           // [ctas] CTAs that have left their part of the request and head whose first part is CTA c's; zero between launches
  uint2* prefix;          // [requests] what lies before a request: tiles, segments
  long long ld_q, ld_out;
  int rows, requests, max_pages, num_pages, page_granules;
  int q_heads, kv_heads, group, max_new;
  float scale_log2, inv_group;
  unsigned long long timeout_ns;
  Status* status;
};

// x / d of small whole numbers (below 2^20) by the reciprocal of d.
__device__ __forceinline__ int div_small(int x, float inv) { return static_cast<int>((static_cast<float>(x) + 0.5f) * inv); }

// What a request adds to the list: segments (a key/value head and set of columns) of `tiles` each.
struct Weight {
  int len, fresh, tiles, blocks;  // blocks: sets of columns (new token x head of the group) of a key/value head
};

template <int COLS>
__device__ __forceinline__ Weight weight_of(const AttnParams& p, int len, int fresh) {
  Weight w;
  w.len = len;
  w.fresh = fresh;
  const int served = min(fresh, p.max_new);
  w.tiles = max((len + TILE - 1) / TILE, 1);  // a row without keys still has its output (zeros) to be written
  w.blocks = served > 0 ? (served * p.group + COLS - 1) / COLS : 0;
  return w;
}
template <int COLS>
__device__ __forceinline__ Weight load_weight(const AttnParams& p, int b) {
  const int len = static_cast<int>(min(static_cast<long long>(max(p.seq_lens[b], 0)), static_cast<long long>(p.max_pages) * p.page_granules * GRANULE));
  return weight_of<COLS>(p, len, p.new_lens != nullptr ? p.new_lens[b] : 1);
}

// The list is cut by cost (tiles and SEGMENT_COST a segment) into parts that differ by one at most. A CTA has work
// for every warp before there is another one.
struct Cut {
  unsigned parts, each, longer;  // the first `longer` parts are each + 1 long, the others each
  __device__ __forceinline__ Cut(unsigned cost, unsigned n) : parts(n), each(cost / n), longer(cost - each * n) {}
  __device__ __forceinline__ unsigned start(unsigned c) const { return each * c + min(c, longer); }
  __device__ __forceinline__ unsigned part_of(unsigned at) const {
    const unsigned head = longer * (each + 1);
    return at < head ? at / (each + 1) : longer + (at - head) / each;
  }
};
__device__ __forceinline__ unsigned cost_of(const uint2& v) { return v.x + SEGMENT_COST * v.y; }

__device__ __forceinline__ float ex2f(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // e in [-126, 127]
__device__ __forceinline__ int exponent_of(float x) { return static_cast<int>((__float_as_uint(x) >> 23) & 0xffu) - 127; }
// A whole number above log2 |x| by one at most: the biased exponent, put behind 2^23.
__device__ __forceinline__ float above_log2(float x) { return __uint_as_float(((__float_as_uint(x) >> 23) & 0xffu) | 0x4b000000u) - (8388608.0f + 126.0f); }

__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// Two pairs of codes of a 32-bit word as fp16 subnormals: n 2^-24 and 16 n 2^-24.
__device__ __forceinline__ uint32_t code_lo(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t code_hi(uint32_t w) { return w & 0x00f000f0u; }

__device__ __forceinline__ float sum_rows(float v) {  // over the 8 lanes that share lane % 4
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}
__device__ __forceinline__ float max_rows(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}

// A tile in the ring. `flags`: tile of the segment << 3, whether a segment begins with it (but for the part's
// first tile), whether each of its granules has a page.
struct Desc {
  int flags, b, hc;  // request, key/value head * blocks + block
};
constexpr int TILE_FIRST = 4, TILE_PAGES = 3;

// What a warp leaves of requests it does not hold whole: `head` began in an earlier warp, `tail` goes on in a later one.
// The last thing that a warp leaves lies in its ring, a head that it goes on from in p.heads.
struct Ends {
  int head_b, head_hc, head_ends;  // head_b < 0: none; head_ends: its last tile is in this warp
  int head_in_ring;
  int tail_b, tail_hc;             // tail_b < 0: none
  int used;                        // whether the warp has tiles
};

// Q^T fragments of a segment, of every lane: the four pairs of each word of its 16 bytes.
template <int NT>
struct Queries {
  uint4 qf[NT][4][32];
};

template <int NT, int WARPS, int STAGES>
struct AttnShared {
  static constexpr int COLS = 8 * NT;
  uint8_t ring[WARPS][STAGES][TILE_BYTES];       // at the end: what a warp leaves
  Desc desc[WARPS][STAGES];
  uint64_t full[WARPS][STAGES];
  uint2 prefix[REQUESTS_IN_SMEM];
  uint2 part[WARPS + 1];                         // first tile of a warp's part and its request
  Queries<NT> queries[WARPS + 1];                // of the warps' segments; the last: of the CTA's first segment
  float2 column[NT][2][32];                      // c1 and sq of the CTA's first segment, of every lane
  int2 lens[REQUESTS_IN_SMEM];                   // length, new tokens
  uint2 warp_sum[WARPS];
  unsigned warp_longest[WARPS];
  Ends ends[WARPS];
  int order[WARPS];                              // the warps that have tiles
  uint32_t abort;
  unsigned cost, parts, whole;                   // the cut: cost of the list, CTAs with work, whether segments stay whole
  int2 joins[2];                                 // first CTA and number of the parts of its first / last segment that this CTA joins
  static_assert(STAGES * TILE_BYTES >= COLS * PARTIAL_FLOATS * 4, "a partial result fits into the ring");
};

// Weighted sum of one column of the partial results `link(i)`, i in [0, n): lane l has dimensions 4l .. 4l + 3.
// Results are relative to the largest reference; `sum` and `ref` are the joined ones. Eight parts are in flight at a time.
template <typename Link>
__device__ __forceinline__ float4 join_links(int n, Link link, int lane, float& sum, float& ref) {
  float best = -INFINITY;
  sum = 0.0f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += 8) {
    float4 v[8];
    float2 ml[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i0 + i < n) {
        const float* s = link(i0 + i);
        v[i] = *reinterpret_cast<const float4*>(s + 4 * lane);
        ml[i] = *reinterpret_cast<const float2*>(s + HEAD_DIM);
      } else {
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        ml[i] = make_float2(0.f, 0.f);
      }
    float top = best;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = ml[i].y != 0.0f ? fmaxf(top, ml[i].x) : top;  // a part without keys has no reference
    const float keep = best == -INFINITY ? 0.0f : ex2f(best - top);
    best = top;
    sum *= keep;
    acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = ml[i].y == 0.0f ? 0.0f : ex2f(ml[i].x - top);
      sum = fmaf(f, ml[i].y, sum);
      acc.x = fmaf(f, v[i].x, acc.x);
      acc.y = fmaf(f, v[i].y, acc.y);
      acc.z = fmaf(f, v[i].z, acc.z);
      acc.w = fmaf(f, v[i].w, acc.w);
    }
  }
  ref = best == -INFINITY ? 0.0f : best;
  return acc;
}
__device__ __forceinline__ void store_row(__nv_bfloat16* dst, float4 v, float sum) {
  const bool any = sum != 0.0f;  // no keys: zeros
  const float inv = 1.0f / sum;
  const __nv_bfloat162 lo = __floats2bfloat162_rn(any ? v.x * inv : 0.f, any ? v.y * inv : 0.f);
  const __nv_bfloat162 hi = __floats2bfloat162_rn(any ? v.z * inv : 0.f, any ? v.w * inv : 0.f);
  *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

// NT: sets of 8 columns a warp carries. One CTA an SM; the registers of a warp decide how many warps it has.
template <int NT, int WARPS, int STAGES>
__global__ void __launch_bounds__(WARPS * 32, 1) attention_paged4_kernel(const AttnParams p) {
  constexpr int COLS = 8 * NT, THREADS = WARPS * 32;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  auto& sm = *reinterpret_cast<AttnShared<NT, WARPS, STAGES>*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  if (lane < STAGES) mbar_init(&sm.full[warp][lane], 1);
  if (threadIdx.x == 0) sm.abort = 0u;
  mbar_fence_init();
  const Deadline dl{globaltimer_ns() + p.timeout_ns, &sm.abort, p.status};
  grid_dependency_wait();
  grid_launch_dependents();

  // ---- prefix sums over the requests (many requests: in the workspace, where every CTA writes the same numbers)
  const bool in_smem = p.requests <= REQUESTS_IN_SMEM;
  uint2* prefix = in_smem ? sm.prefix : p.prefix;
  uint2 all{0, 0};
  unsigned longest = 0;  // tiles
  auto take_in = [&](int b) {  // a request's tiles and segments
    uint2 v{0, 0};
    if (b < p.requests) {
      const Weight w = load_weight<COLS>(p, b);
      v.y = static_cast<unsigned>(w.blocks) * p.kv_heads;
      v.x = v.y * w.tiles;
      if (in_smem) sm.lens[b] = make_int2(w.len, w.fresh);
      if (w.blocks > 0) longest = max(longest, static_cast<unsigned>(w.tiles));
    }
    return v;
  };
  auto scan = [&](uint2 v) {  // sums over this lane and those before it
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned ux = __shfl_up_sync(0xffffffffu, v.x, o), uy = __shfl_up_sync(0xffffffffu, v.y, o);
      if (lane >= o) {
        v.x += ux;
        v.y += uy;
      }
    }
    return v;
  };
  if (p.requests <= 4 * 32) {  // one warp, four requests a lane
    if (warp == 0) {
      uint2 v[4], own{0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = take_in(4 * lane + i);
        own.x += v[i].x;
        own.y += v[i].y;
      }
      const uint2 inc = scan(own);
      uint2 before = make_uint2(inc.x - own.x, inc.y - own.y);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (4 * lane + i < p.requests) prefix[4 * lane + i] = before;
        before.x += v[i].x;
        before.y += v[i].y;
      }
      longest = __reduce_max_sync(0xffffffffu, longest);
      all = make_uint2(__shfl_sync(0xffffffffu, inc.x, 31), __shfl_sync(0xffffffffu, inc.y, 31));
      __syncwarp();
    }
  } else {
    for (int b0 = 0; b0 < p.requests; b0 += THREADS) {
      const int b = b0 + threadIdx.x;
      const uint2 v = take_in(b), inc = scan(v);
      if (b0 > 0) __syncthreads();
      longest = __reduce_max_sync(0xffffffffu, longest);
      if (lane == 31) {
        sm.warp_sum[warp] = inc;
        sm.warp_longest[warp] = longest;
      }
      __syncthreads();
      uint2 before = all;
      const int holding = min(WARPS, (p.requests - b0 + 31) >> 5);  // warps with a request
      for (int i = 0; i < holding; ++i) {
        const uint2 s = sm.warp_sum[i];
        longest = max(longest, sm.warp_longest[i]);
        if (i < warp) {
          before.x += s.x;
          before.y += s.y;
        }
        all.x += s.x;
        all.y += s.y;
      }
      if (b < p.requests) prefix[b] = make_uint2(before.x + inc.x - v.x, before.y + inc.y - v.y);
    }
    __syncthreads();
  }

  auto weight = [&](int b) { return in_smem ? weight_of<COLS>(p, sm.lens[b].x, sm.lens[b].y) : load_weight<COLS>(p, b); };
  auto cut_of = [&](unsigned cost) { return Cut(cost, min(static_cast<unsigned>(gridDim.x), (cost + WARPS - 1) / WARPS)); };
  if (warp == 0) {
    const unsigned cost = cost_of(all);
    unsigned parts = 0, per_cta = 1;
    bool whole = false;
    if (cost > 0) {
      const Cut cut = cut_of(cost);
      // Whole segments a CTA where that costs less than the joins that it saves (128 requests of 4096 tokens, one key/value
      // head, on 148 CTAs: 24.8 us against 27.3 us cut evenly)
      per_cta = (all.y + gridDim.x - 1) / gridDim.x;
      whole = per_cta * (longest + SEGMENT_COST) <= cut.each + JOIN_COST / NT;
      parts = whole ? (all.y + per_cta - 1) / per_cta : cut.parts;
      if (blockIdx.x < parts) {
        // the last request for which `before` (of what lies before it) is at most x: it is not empty
        auto find = [&](unsigned x, auto before) {
          int lo = 0, hi = p.requests;
          while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (before(prefix[mid]) <= x) lo = mid; else hi = mid;
          }
          return lo;
        };
        auto part_start = [&](unsigned c) {
          if (!whole) return cut.start(c);
          const unsigned s = c * per_cta;
          if (s >= all.y) return cost;
          const int b = find(s, [](const uint2& v) { return v.y; });
          return cost_of(prefix[b]) + (s - prefix[b].y) * (static_cast<unsigned>(weight(b).tiles) + SEGMENT_COST);
        };
        // The parts of this CTA's warps, cut by cost too: lane w finds where warp w's begins. (Every warp has the queries of
        // its first segment to fetch: the CTA's first segment costs nothing more.)
        const unsigned bound = part_start(blockIdx.x + (lane & 1));
        const unsigned at0 = __shfl_sync(0xffffffffu, bound, 0) + (whole ? SEGMENT_COST : 0u), at_n = __shfl_sync(0xffffffffu, bound, 1) - at0;
        const unsigned at = at0 + Cut(at_n, WARPS).start(min(lane, WARPS));
        uint2 begin{all.x, 0u};  // tiles that lie before that place, and the request that it is in
        if (at < cost) {
          const int b = find(at, [](const uint2& v) { return cost_of(v); });
          const unsigned tiles = weight(b).tiles, rel = at - cost_of(prefix[b]), each = tiles + SEGMENT_COST;
          const unsigned s = rel / each, in = rel - s * each;
          begin = make_uint2(prefix[b].x + s * tiles + (in > SEGMENT_COST ? in - SEGMENT_COST : 0u), static_cast<unsigned>(b));
        }
        if (lane <= WARPS) sm.part[lane] = begin;
      }
    }
    if (lane == 0) {
      sm.cost = cost;
      sm.parts = parts;
      sm.whole = whole;
      sm.joins[0] = sm.joins[1] = make_int2(0, 0);
    }
  }
  __syncthreads();
  if (blockIdx.x >= sm.parts) return;
  const bool whole = sm.whole != 0u;
  const unsigned f0 = sm.part[warp].x;
  const int count = static_cast<int>(sm.part[warp + 1].x - f0);
  int cur_b = static_cast<int>(sm.part[warp].y);  // request of the part's first tile, then of the last look-up's first
  auto request_of = [&](int b, unsigned f) {  // of tile f, from a request at or before it
    while (b + 1 < p.requests && prefix[b + 1].x <= f) ++b;
    return b;
  };

  // ---- copies: lane i looks up the i-th of the next 32 tiles; `issue(s)` starts the copies of its tile into stage s
  Desc ahead{0, 0, 0};
  const uint8_t* ahead_src[2] = {nullptr, nullptr};
  auto look_up = [&](int n) {
    cur_b = request_of(cur_b, f0 + n);
    if (n + lane < count) {
      const unsigned f = f0 + n + lane;
      const int b = request_of(cur_b, f);
      const Weight w = weight(b);
      const unsigned rel = f - prefix[b].x, hc = rel / w.tiles;
      const int tile = static_cast<int>(rel - hc * w.tiles);
      ahead.b = b;
      ahead.hc = static_cast<int>(hc);
      ahead.flags = tile << 3 | (tile == 0 && n + lane > 0 ? TILE_FIRST : 0);
      const int kvh = w.blocks == 1 ? ahead.hc : ahead.hc / w.blocks;
      int column = 2 * tile / p.page_granules, in_page = 2 * tile - column * p.page_granules;  // the length keeps it inside the table
      const int* row = p.table + static_cast<size_t>(b) * p.max_pages;
      const int page0 = w.len > 0 ? row[column] : -1;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if ((2 * tile + h) * GRANULE >= w.len) break;
        if (h == 1 && ++in_page == p.page_granules) {
          in_page = 0;
          ++column;
        }
        const int page = h == 1 && in_page == 0 ? row[column] : page0;
        if (page >= 0 && page < p.num_pages) {
          ahead.flags |= 1 << h;
          ahead_src[h] = p.cache + ((static_cast<size_t>(page) * p.kv_heads + kvh) * p.page_granules + in_page) * GRANULE_BYTES;
        }
      }
    }
  };
  auto issue = [&](int s) {  // by the lane that looked the tile up
    sm.desc[warp][s] = ahead;
    uint8_t* dst = sm.ring[warp][s];
    uint64_t* bar = &sm.full[warp][s];
    if ((ahead.flags & TILE_PAGES) == TILE_PAGES && ahead_src[1] == ahead_src[0] + GRANULE_BYTES) {
      mbar_expect_tx(bar, TILE_BYTES);
      bulk_load(dst, ahead_src[0], TILE_BYTES, bar);
    } else {  // a page ends in the middle, or what is not there is not copied: its keys are masked
      const int halves = (ahead.flags & 1) + (ahead.flags >> 1 & 1);
      if (halves == 0) mbar_arrive(bar);
      else mbar_expect_tx(bar, halves * GRANULE_BYTES);
      if ((ahead.flags & 1) != 0) bulk_load(dst, ahead_src[0], GRANULE_BYTES, bar);
      if ((ahead.flags & 2) != 0) bulk_load(dst + GRANULE_BYTES, ahead_src[1], GRANULE_BYTES, bar);
    }
  };

  // ---- state of the segment (one request, key/value head and set of columns)
  uint4 qf[NT == 1 ? 4 : 1];                  // Q^T fragments; with two sets of columns they stay in shared memory
  int query_slot = warp;
  float c1[NT][2], sq[NT][2];                 // score = (acc s_k + sq m_k) c1, of columns 2t and 2t + 1
  int limit[NT][2];                           // keys a column sees
  float ref[NT][2], over[NT][2];              // reference (log2); a score that exceeds it by `over` moves it (-inf: none yet)
  float l[NT][2], pm[NT][2];                  // sum p and sum p (m_v + 7.5 s_v), of this thread's keys
  float acc[NT][8][4];
  float tilt[NT][4];                          // what keys 0-7 of the granules weigh more than keys 8-15, since acc was levelled
  float f[NT][2], w_limit[NT][2];             // p s_v is held times f = 2^e; what exceeds 2^w_limit, w_limit = 15 - e, moves it
  int seg_b = -1, seg_hc = 0, seg_first = 0, seg_last = 0, min_limit = 0;
  Ends ends{-1, -1, 0, 0, -1, -1, count > 0 ? 1 : 0};

  // head, first column and first row of a segment
  auto place = [&](const Weight& w, int b, int hc, int& kvh, int& column0, int& row0) {
    kvh = w.blocks == 1 ? hc : hc / w.blocks;
    column0 = (hc - kvh * w.blocks) * COLS;
    row0 = p.row_starts != nullptr ? p.row_starts[b] : b;
  };

  uint4 raw[NT][4];
  auto load_queries = [&](int b, int hc) {  // this lane's 32 dimensions of column g of each set
    const Weight w = weight(b);
    int kvh, column0, row0;
    place(w, b, hc, kvh, column0, row0);
    const int served = min(w.fresh, p.max_new);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int c = column0 + nt * 8 + g, j = div_small(c, p.inv_group), row = row0 + j;
      const bool here = j < served && row >= 0 && row < p.rows;
      const __nv_bfloat16* src = p.q + row * p.ld_q + (kvh * p.group + c - j * p.group) * HEAD_DIM + t * 32;
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[nt][i] = here ? *reinterpret_cast<const uint4*>(src + i * 8) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  auto make_fragments = [&](int slot) {  // from the queries that were loaded
    auto& to = sm.queries[slot];
    query_slot = slot;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[32], big = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w4[4] = {raw[nt][i].x, raw[nt][i].y, raw[nt][i].z, raw[nt][i].w};
        float most = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[i * 8 + 2 * k] = __uint_as_float(w4[k] << 16);
          x[i * 8 + 2 * k + 1] = __uint_as_float(w4[k] & 0xffff0000u);
          most = fmaxf(fmaxf(most, fabsf(x[i * 8 + 2 * k])), fabsf(x[i * 8 + 2 * k + 1]));
        }
        big = fmaxf(big, most);
      }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      const int e = max(min(exponent_of(big), 117), -100);
      const float up[2] = {pow2i(14 - e), pow2i(10 - e)};
      uint32_t f[16];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // word i of the 16 bytes, nibbles k and k + 4: dimensions 8i + k and 8i + k + 4 (odd k: 16 times the code)
          const __half2 h = __floats2half2_rn(x[i * 8 + k] * up[k & 1], x[i * 8 + k + 4] * up[k & 1]);
          f[i * 4 + k] = *reinterpret_cast<const uint32_t*>(&h);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) to.qf[nt][i][lane] = make_uint4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
      // the sum of q: its product with codes that are all one
      float one[4];
      mma_f16_first(one, 0x00010001u, 0x00010001u, 0x00100010u, 0x00100010u, f[0], f[1]);
#pragma unroll
      for (int i = 1; i < 8; ++i) mma_f16(one, 0x00010001u, 0x00010001u, 0x00100010u, 0x00100010u, f[2 * i], f[2 * i + 1]);
      const float a = p.scale_log2 * pow2i(e + 10);  // 2^24 of the codes, 2^(e - 14) of q
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        c1[nt][k] = __shfl_sync(0xffffffffu, a, (2 * t + k) * 4);  // the columns of this thread's scores: held by lane group 2t + k
        sq[nt][k] = one[k];
      }
    }
    __syncwarp();
  };
  auto hold_fragments = [&]() {
    if (NT == 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) qf[i < NT * 4 ? i : 0] = sm.queries[query_slot].qf[0][i][lane];
  };
  auto begin = [&](int b, int hc, int tile) {  // everything of a segment's state but the fragments
    seg_b = b;
    seg_hc = hc;
    seg_first = tile;
    const Weight w = weight(b);
    int kvh, column0, row0;
    place(w, b, hc, kvh, column0, row0);
    const int served = min(w.fresh, p.max_new);
    min_limit = w.len;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int j = div_small(column0 + nt * 8 + 2 * t + k, p.inv_group);
        limit[nt][k] = j < served ? min(w.len - w.fresh + j + 1, w.len) : w.len;  // a column without a query is computed and dropped
        ref[nt][k] = 0.f;
        over[nt][k] = -INFINITY;
        f[nt][k] = pow2i(WEIGHT_SCALE_MAX);
        w_limit[nt][k] = WEIGHT_LIMIT - WEIGHT_SCALE_MAX;
        l[nt][k] = 0.f;
        pm[nt][k] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[nt][i][k] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) tilt[nt][k] = 0.f;
      min_limit = min(min_limit, min(limit[nt][0], limit[nt][1]));
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) min_limit = min(min_limit, __shfl_xor_sync(0xffffffffu, min_limit, o));
  };

  // Counts the codes of what is summed from 7.5: keys 0-7 stand there with n, keys 8-15 with n - 15.
  auto level = [&]() {
    constexpr float LO = 7.5f / 16777216.0f, HI = 16.0f * LO;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[nt][i][k] = fmaf(tilt[nt][k & 1], k < 2 ? -LO : -HI, acc[nt][i][k]);
#pragma unroll
      for (int k = 0; k < 4; ++k) tilt[nt][k] = 0.f;
    }
  };

  auto flush = [&](bool last) {
    level();
    const Weight w = weight(seg_b);
    const bool began = seg_first == 0, ended = seg_last == w.tiles - 1;
    int kvh, column0, row0;
    place(w, seg_b, seg_hc, kvh, column0, row0);
    const int served = min(w.fresh, p.max_new);
    float* part = nullptr;
    if (!began || !ended) {
      part = last ? reinterpret_cast<float*>(sm.ring[warp][0])  // every copy into the ring has been read
                  : p.heads + (static_cast<size_t>(blockIdx.x) * WARPS + warp) * COLS * PARTIAL_FLOATS;
      if (!began) {
        ends.head_b = seg_b;
        ends.head_hc = seg_hc;
        ends.head_ends = ended;
        ends.head_in_ring = last;
      } else {
        ends.tail_b = seg_b;
        ends.tail_hc = seg_hc;
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float sum = sum_rows(l[nt][k]), add = sum_rows(pm[nt][k]);
        const int local = nt * 8 + 2 * t + k, c = column0 + local;
        const int j = div_small(c, p.inv_group), row = row0 + j;
        if (j >= served || row < 0 || row >= p.rows) continue;
        const float inv = part != nullptr ? 1.0f : (sum != 0.0f ? 1.0f / sum : 0.0f);  // no keys: zeros
        const float back = pow2i(-exponent_of(f[nt][k])) * inv, more = add * inv;
        float* dst = part + local * PARTIAL_FLOATS;
        __nv_bfloat16* out = p.out + row * p.ld_out + (kvh * p.group + c - j * p.group) * HEAD_DIM;
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
          // dimensions 32 c4 + 4 g .. + 3: rows g and g + 8 of m-tiles 2 c4 and 2 c4 + 1
          constexpr float LO = 0x1p24f, HI = 0x1p20f;  // of the codes
          const float o0 = fmaf(acc[nt][2 * c4][k] * LO, back, more), o1 = fmaf(acc[nt][2 * c4][2 + k] * HI, back, more);
          const float o2 = fmaf(acc[nt][2 * c4 + 1][k] * LO, back, more), o3 = fmaf(acc[nt][2 * c4 + 1][2 + k] * HI, back, more);
          const int dim = 32 * c4 + 4 * g;
          if (part == nullptr) {
            const __nv_bfloat162 lo = __floats2bfloat162_rn(o0, o1), hi = __floats2bfloat162_rn(o2, o3);
            *reinterpret_cast<uint2*>(out + dim) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
          } else {
            *reinterpret_cast<float4*>(dst + dim) = make_float4(o0, o1, o2, o3);
          }
        }
        if (part != nullptr && g == 0) *reinterpret_cast<float2*>(dst + HEAD_DIM) = make_float2(ref[nt][k], sum);
      }
  };

  // lane's row address of the transposed loads: matrix lane / 8 of four (keys 0-7 / 8-15 of chunks c, c + 1)
  const int lm_row = (lane & 7) + ((lane >> 3) & 1) * 8;
  const uint32_t lm_off = HALF_GRANULE + lm_row * CODE_BYTES + (chunk_place(lane >> 4, lm_row) << 4);
  const uint32_t k_off = g * CODE_BYTES + (chunk_place(t, g) << 4);

  // The first queries are on their way while the pages are looked up and the first copies start. Warps that begin in the
  // CTA's first segment (all of them where requests are long) take its fragments from the first warp.
  int first_b = 0, first_hc = 0, first_tile = 0;
  bool shared_queries = false;
  if (count > 0) {
    first_b = cur_b = request_of(cur_b, f0);
    const unsigned tiles = weight(first_b).tiles, rel = f0 - prefix[first_b].x;
    first_hc = static_cast<int>(rel / tiles);
    first_tile = static_cast<int>(rel) - first_hc * static_cast<int>(tiles);
    shared_queries = warp > 0 && f0 - first_tile <= sm.part[0].x && sm.part[1].x > sm.part[0].x;  // the segment began at or before the CTA's first tile
    if (!shared_queries) load_queries(first_b, first_hc);
    look_up(0);
    if (lane < STAGES && lane < count) issue(lane);
    __syncwarp();
    begin(first_b, first_hc, first_tile);
    if (!shared_queries) make_fragments(warp == 0 ? WARPS : warp);
    if (warp == 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) sm.column[nt][k][lane] = make_float2(c1[nt][k], sq[nt][k]);
    }
  }
  __syncthreads();
  if (shared_queries) {
    query_slot = WARPS;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float2 v = sm.column[nt][k][lane];
        c1[nt][k] = v.x;
        sq[nt][k] = v.y;
      }
  }
  hold_fragments();
  bool ok = true;
  int stage = 0, phase = 0, base = 0;  // ring position of tile n; first tile of the last look-up
  for (int n = 0; n < count; ++n) {
    const int flags = sm.desc[warp][stage].flags, tile = flags >> 3;
    if ((flags & TILE_FIRST) != 0) {
      flush(false);
      load_queries(sm.desc[warp][stage].b, sm.desc[warp][stage].hc);
      make_fragments(warp);
      hold_fragments();
      begin(sm.desc[warp][stage].b, sm.desc[warp][stage].hc, tile);
    }
    seg_last = tile;
    const bool there = mbar_try_wait(&sm.full[warp][stage], phase);
    if (!__all_sync(0xffffffffu, there)) {
      ok = mbar_wait(&sm.full[warp][stage], phase, dl, WHERE_PAGED_ATTN, blockIdx.x);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
    }
    const uint8_t* st = sm.ring[warp][stage];
    const bool edge = (flags & TILE_PAGES) != TILE_PAGES || (tile + 1) * TILE > min_limit;

    // ---- S^T = K Q^T
    float sc[2][NT][4];
    {
      uint4 ka[2], kb[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ka[h] = *reinterpret_cast<const uint4*>(st + h * GRANULE_BYTES + k_off);
        kb[h] = *reinterpret_cast<const uint4*>(st + h * GRANULE_BYTES + k_off + 8 * CODE_BYTES);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4 q[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) q[nt] = NT == 1 ? qf[NT == 1 ? i : 0] : sm.queries[query_slot].qf[nt][i][lane];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t wa = i == 0 ? ka[h].x : i == 1 ? ka[h].y : i == 2 ? ka[h].z : ka[h].w;
          const uint32_t wb = i == 0 ? kb[h].x : i == 1 ? kb[h].y : i == 2 ? kb[h].z : kb[h].w;
          const uint32_t a8 = wa >> 8, b8 = wb >> 8;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (i == 0) mma_f16_first(sc[h][nt], code_lo(wa), code_lo(wb), code_hi(wa), code_hi(wb), q[nt].x, q[nt].y);
            else mma_f16(sc[h][nt], code_lo(wa), code_lo(wb), code_hi(wa), code_hi(wb), q[nt].x, q[nt].y);
            mma_f16(sc[h][nt], code_lo(a8), code_lo(b8), code_hi(a8), code_hi(b8), q[nt].z, q[nt].w);
          }
        }
      }
    }
    // with registers to spare the value fragments are on their way while the softmax works
    constexpr bool EARLY = NT == 2;
    uint32_t vf[2][2][4];  // (keys 0-7, keys 8-15) of chunk 2 half, then of chunk 2 half + 1
    auto load_values = [&](int h, int half) { ldmatrix_x4_trans(smem_u32(st) + h * GRANULE_BYTES + (lm_off ^ (half * 32)), vf[h][half]); };
    if (EARLY) {
#pragma unroll
      for (int i = 0; i < 4; ++i) load_values(i >> 1, i & 1);
    }
    // ---- scores less their reference, log2
    float vs[2][2], vm[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t kp = *reinterpret_cast<const uint32_t*>(st + h * GRANULE_BYTES + PARAM_OFFSET + (g + 8 * r) * 4);
        const uint32_t vp = *reinterpret_cast<const uint32_t*>(st + h * GRANULE_BYTES + HALF_GRANULE + PARAM_OFFSET + (g + 8 * r) * 4);
        const float ks = __uint_as_float(kp << 16), km = __uint_as_float(kp & 0xffff0000u);
        vs[h][r] = __uint_as_float(vp << 16);
        vm[h][r] = __uint_as_float(vp & 0xffff0000u);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float& x = sc[h][nt][2 * r + c];
            x = fmaf(fmaf(x, ks, sq[nt][c] * km), c1[nt][c], -ref[nt][c]);
          }
      }
    if (edge) {  // masked keys: no score, and parameters (whatever lies there) that count for nothing
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const bool page = (flags >> h & 1) != 0;
          const int key = tile * TILE + h * GRANULE + g + 8 * r;
          bool any = false, seen[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              seen[nt][c] = page && key < limit[nt][c];
              any = any || seen[nt][c];
              if (!seen[nt][c]) sc[h][nt][2 * r + c] = -INFINITY;
            }
          if (!any) {
            vs[h][r] = vm[h][r] = 0.f;
          } else if (!(fabsf(vs[h][r]) + fabsf(vm[h][r]) < INFINITY)) {
            // parameters that are no numbers must not meet the weight 0 of a column that does not see the key: the
            // columns that see it take the NaN through their sum
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 2; ++c)
                if (seen[nt][c]) l[nt][c] = NAN;
            vs[h][r] = vm[h][r] = 0.f;
          }
        }
    }
    // from here on the middle of a token's values instead of their minimum
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 2; ++r) vm[h][r] = fmaf(7.5f, vs[h][r], vm[h][r]);
    // What may move a column's references: a score above them, or a score and a scale (of one key, or so it is assumed here)
    const float vmax = fmaxf(fmaxf(fabsf(vs[0][0]), fabsf(vs[0][1])), fmaxf(fabsf(vs[1][0]), fabsf(vs[1][1])));
    const float vtop = above_log2(vmax);
    float top[NT][2];
    bool move = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[nt][c] = fmaxf(fmaxf(sc[0][nt][c], sc[0][nt][2 + c]), fmaxf(sc[1][nt][c], sc[1][nt][2 + c]));
        move = move || top[nt][c] > fminf(over[nt][c], w_limit[nt][c] - vtop);
      }
    if (__any_sync(0xffffffffu, move)) {
      // new references: of p the largest score of each column so far, of p s_v f what the largest p s_v so far asks for. f stays a
      // whole power of two: the largest p is 1, and its weight is not rounded.
      float ev[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r) ev[h][r] = above_log2(vs[h][r]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const bool none = over[nt][c] == -INFINITY;  // no key so far
          const float high = max_rows(top[nt][c]), up = none ? high : fmaxf(high, 0.0f);
          const float rise = up != -INFINITY ? up : 0.0f;
          const float weighted = max_rows(fmaxf(fmaxf(sc[0][nt][c] + ev[0][0], sc[0][nt][2 + c] + ev[0][1]), fmaxf(sc[1][nt][c] + ev[1][0], sc[1][nt][2 + c] + ev[1][1])));
          // f = 2^-e, no smaller an exponent than the sums now have relative to the new reference
          const float now = none ? -WEIGHT_SCALE_MAX : w_limit[nt][c] - WEIGHT_LIMIT - rise;
          const float e = ceilf(fmaxf(fmaxf(now, -WEIGHT_SCALE_MAX), weighted - rise - WEIGHT_TOP));
          const float alpha = none ? 1.0f : ex2f(-rise), beta = none ? 1.0f : ex2f(now - e);
          if (up != -INFINITY) over[nt][c] = RESCALE_LIMIT;
          ref[nt][c] += rise;
          l[nt][c] *= alpha;
          pm[nt][c] *= alpha;
          f[nt][c] = pow2i(-static_cast<int>(e));
          w_limit[nt][c] = WEIGHT_LIMIT + e;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            acc[nt][i][c] *= beta;
            acc[nt][i][2 + c] *= beta;
          }
          tilt[nt][c] *= beta;
          tilt[nt][2 + c] = 0.f;  // the rows are all alike, these are not read
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            sc[h][nt][c] -= rise;
            sc[h][nt][2 + c] -= rise;
          }
        }
    }
    // ---- P^T, then O^T += V^T P^T
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t pf[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = k >> 1, c = k & 1;
          const float pr = ex2f(sc[h][nt][k]);
          l[nt][c] += pr;
          w[k] = pr * (r == 0 ? f[nt][c] : -f[nt][c]) * vs[h][r];
          pm[nt][c] = fmaf(pr, vm[h][r], pm[nt][c]);
        }
        const __half2 h0 = __floats2half2_rn(w[0], w[1]), h1 = __floats2half2_rn(w[2], w[3]);
        pf[nt][0] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h0));
        pf[nt][1] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h1));
        mma_f16(tilt[nt], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, pf[nt][0], pf[nt][1]);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (!EARLY) load_values(h, half);
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          const uint32_t x0 = vf[h][half][2 * cc], x1 = ~vf[h][half][2 * cc + 1], y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(acc[nt][4 * half + 2 * cc], code_lo(x0), code_hi(x0), code_lo(x1), code_hi(x1), pf[nt][0], pf[nt][1]);
            mma_f16(acc[nt][4 * half + 2 * cc + 1], code_lo(y0), code_hi(y0), code_lo(y1), code_hi(y1), pf[nt][0], pf[nt][1]);
          }
        }
      }
    }
    if ((n & (LEVEL_TILES - 1)) == LEVEL_TILES - 1) level();
    __syncwarp();  // every lane has read the stage
    const int next = n + STAGES;
    if (next < count) {
      if (next - base == 32) look_up(base = next);
      if (lane == next - base) issue(stage);
      __syncwarp();
    }
    if (++stage == STAGES) {
      stage = 0;
      phase ^= 1;
    }
  }
  if (ok) {
    __syncwarp();
    if (count > 0) flush(true);
  } else {
    // a wait ran out: this warp's copies may still be on their way into shared memory
    const uint64_t t_stop = globaltimer_ns() + 2000000ull;
    while (globaltimer_ns() < t_stop) __nanosleep(1000);
  }
  if (lane == 0) sm.ends[warp] = ends;
  __syncthreads();

  // ---- what is cut between warps: a chain begins with a warp's tail (or with the first warp's head, which began in the
  // CTA before) and goes through the heads of the following warps. One warp a chain and column.
  const unsigned used = __ballot_sync(0xffffffffu, lane < WARPS && sm.ends[lane < WARPS ? lane : 0].used != 0);
  const int active = __popc(used);
  if (lane < WARPS && (used >> lane & 1u) != 0u) sm.order[__popc(used & ((1u << lane) - 1u))] = lane;  // every warp writes the same
  __syncwarp();
  if (active == 0) return;
  const unsigned tails = __ballot_sync(0xffffffffu, lane < active && sm.ends[sm.order[lane < active ? lane : 0]].tail_b >= 0);
  const int before = sm.ends[sm.order[0]].head_b >= 0 ? 1 : 0, chains = before + __popc(tails);
  if (chains == 0) return;
  const unsigned ending = __ballot_sync(0xffffffffu, lane < active && sm.ends[sm.order[lane < active ? lane : 0]].head_ends != 0);
  // lane k has chain k: where it begins (place among the warps with work of the one with its tail, -1: the first one's
  // head), its links, and what its rows are
  int ch_b = 0, ch_hc = 0, ch_start = -1, ch_links = 0, ch_head = 0, ch_column0 = 0, ch_row0 = 0, ch_served = 0;
  bool ch_ended = false;
  if (lane < chains) {
    unsigned later = tails;
    for (int i = before; i < lane; ++i) later &= later - 1u;
    if (lane >= before) ch_start = __ffs(later) - 1;
    const Ends& e = sm.ends[sm.order[max(ch_start, 0)]];
    ch_b = ch_start < 0 ? e.head_b : e.tail_b;
    ch_hc = ch_start < 0 ? e.head_hc : e.tail_hc;
    const unsigned ends = ending >> (ch_start + 1);  // the first of the following heads that ends (at most 16 warps)
    ch_ended = ends != 0u;
    ch_links = (ch_ended ? ch_start + 1 + __ffs(ends) : active) - max(ch_start, 0);
    const Weight w = weight(ch_b);
    place(w, ch_b, ch_hc, ch_head, ch_column0, ch_row0);
    ch_head *= p.group;
    ch_served = min(w.fresh, p.max_new);
  }
  const int columns = min(COLS, p.max_new * p.group);  // of a segment with queries, at most
  for (int task = warp; task < chains * columns; task += WARPS) {
    const int k = task / columns, local = task - k * columns;
    const int start = __shfl_sync(0xffffffffu, ch_start, k), links = __shfl_sync(0xffffffffu, ch_links, k);
    const int c = __shfl_sync(0xffffffffu, ch_column0, k) + local, j = div_small(c, p.inv_group);
    const int row = __shfl_sync(0xffffffffu, ch_row0, k) + j, head = __shfl_sync(0xffffffffu, ch_head, k) + c - j * p.group;
    const bool ended = __shfl_sync(0xffffffffu, ch_ended, k), here = j < __shfl_sync(0xffffffffu, ch_served, k);
    if (!here || row < 0 || row >= p.rows) continue;
    auto link = [&](int i) -> const float* {
      const int w = sm.order[max(start, 0) + i];
      const bool in_ring = (start >= 0 && i == 0) || sm.ends[w].head_in_ring != 0;
      return (in_ring ? reinterpret_cast<const float*>(sm.ring[w][0]) : p.heads + (static_cast<size_t>(blockIdx.x) * WARPS + w) * COLS * PARTIAL_FLOATS) + local * PARTIAL_FLOATS;
    };
    float sum, joined;
    const float4 v = join_links(links, link, lane, sum, joined);
    if (start >= 0 && ended) {
      store_row(p.out + row * p.ld_out + head * HEAD_DIM + 4 * lane, v, sum);
    } else {
      float* slot = p.partial + ((static_cast<size_t>(blockIdx.x) * 2 + (start >= 0 ? 1 : 0)) * COLS + local) * PARTIAL_FLOATS;
      *reinterpret_cast<float4*>(slot + 4 * lane) = v;
      if (lane == 0) *reinterpret_cast<float2*>(slot + HEAD_DIM) = make_float2(joined, sum);
    }
  }

  if (whole) return;
  // ---- what is cut between CTAs: the first chain if it began in an earlier CTA, the last one if it goes on
  __syncthreads();
  if (warp == 0 && lane < chains && ((lane == 0 && ch_start < 0) || (lane == chains - 1 && ch_start >= 0 && !ch_ended))) {
    // the CTAs that hold tiles of the segment
    const Cut cut = cut_of(sm.cost);
    const unsigned tiles = weight(ch_b).tiles, at = cost_of(prefix[ch_b]) + ch_hc * (tiles + SEGMENT_COST) + SEGMENT_COST;
    const int c0 = static_cast<int>(cut.part_of(at)), n = static_cast<int>(cut.part_of(at + tiles - 1)) - c0 + 1;
    int before_me;  // releases what the other warps wrote before the barrier, acquires what the other CTAs released
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before_me) : "l"(p.arrived + c0) : "memory");
    if (before_me == n - 1) {
      p.arrived[c0] = 0;  // nobody else comes in this launch
      sm.joins[ch_start < 0 ? 0 : 1] = make_int2(c0, n);
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const int c0 = sm.joins[k].x, n = sm.joins[k].y;
    if (n == 0) continue;
    const int chain = k == 0 ? 0 : chains - 1;
    const int column0 = __shfl_sync(0xffffffffu, ch_column0, chain), row0 = __shfl_sync(0xffffffffu, ch_row0, chain);
    const int head0 = __shfl_sync(0xffffffffu, ch_head, chain), served = __shfl_sync(0xffffffffu, ch_served, chain);
    // several warps a column if there are many parts; what they join lies in the rings until one of them joins that
    const int share = n > 8 ? max(WARPS / columns, 1) : 1;
    auto finish = [&](int local, float4 v, float sum) {
      const int c = column0 + local, j = div_small(c, p.inv_group), row = row0 + j;
      if (j < served && row >= 0 && row < p.rows) store_row(p.out + row * p.ld_out + (head0 + c - j * p.group) * HEAD_DIM + 4 * lane, v, sum);
    };
    for (int task = warp; task < columns * share; task += WARPS) {
      const int local = task / share, q = task - local * share, i0 = n * q / share, i1 = n * (q + 1) / share;
      if (div_small(column0 + local, p.inv_group) >= served) continue;  // no query, no part
      auto link = [&](int i) -> const float* { return p.partial + ((static_cast<size_t>(c0 + i0 + i) * 2 + (i0 + i == 0 ? 1 : 0)) * COLS + local) * PARTIAL_FLOATS; };
      float sum, joined;
      const float4 v = join_links(i1 - i0, link, lane, sum, joined);
      if (share == 1) {
        finish(local, v, sum);
      } else {
        float* slot = reinterpret_cast<float*>(sm.ring[warp][0]);
        *reinterpret_cast<float4*>(slot + 4 * lane) = v;
        if (lane == 0) *reinterpret_cast<float2*>(slot + HEAD_DIM) = make_float2(joined, sum);
      }
    }
    if (share > 1) {  // columns * share warps, a task each
      __syncthreads();
      if (warp < columns && div_small(column0 + warp, p.inv_group) < served) {
        auto link = [&](int i) -> const float* { return reinterpret_cast<const float*>(sm.ring[warp * share + i][0]); };
        float sum, joined;
        const float4 v = join_links(share, link, lane, sum, joined);
        finish(warp, v, sum);
      }
      __syncthreads();
    }
  }
}

}  // namespace paged
}  // namespace df

namespace df {
namespace paged {

// Columns (new token x head of the group) of a key/value head that a warp carries: 8 with 16 warps an SM, or 16 with
// 8 warps. 16 read the cache once where 8 would read it twice; 8 or fewer columns have no use for the second set.
constexpr int ATTN_MAX_CTAS = 160;
constexpr int attn_columns(long long columns) { return columns <= 8 ? 8 : 16; }
constexpr int attn_warps(int cols) { return cols == 8 ? 16 : 8; }
constexpr size_t attn_counter_bytes() { return ATTN_MAX_CTAS * sizeof(int); }
static_assert(attn_counter_bytes() == DF_ATTENTION_PAGED4_COUNTER_BYTES, "the public header's number");

template <int NT, int WARPS, int STAGES>
int launch_attention(const AttnParams& p, int grid, cudaStream_t s) {
  using Shared = AttnShared<NT, WARPS, STAGES>;
  static_assert(sizeof(Shared) <= 227 * 1024, "shared memory of an SM");
  auto kernel = attention_paged4_kernel<NT, WARPS, STAGES>;
  static bool attr_set[64] = {false};
  int dev = 0;
  (void)cudaGetDevice(&dev);
  cudaError_t e = cudaSuccess;
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared));
    if (e != cudaSuccess) return fail(DF_ECUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(WARPS * 32, 1, 1);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  cfg.numAttrs = dependent_launch_attr(&attr);
  cfg.attrs = &attr;
  e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(DF_ECUDA, "paged attention launch: %s", cudaGetErrorString(e));
  }
  return DF_OK;
}

}  // namespace paged
}  // namespace df

extern "C" size_t df_attention_paged4_workspace_bytes(int requests, int q_heads, int kv_heads, int max_new) {
  using namespace df::paged;
  if (requests <= 0 || q_heads <= 0 || kv_heads <= 0 || max_new <= 0 || q_heads % kv_heads != 0) return 0;
  const int cols = attn_columns(static_cast<long long>(max_new) * (q_heads / kv_heads));
  const size_t partial = static_cast<size_t>(ATTN_MAX_CTAS) * (2 + attn_warps(cols)) * cols * PARTIAL_FLOATS * sizeof(float);
  return attn_counter_bytes() + static_cast<size_t>(requests + 1) / 2 * 2 * sizeof(uint2) + partial;
}

extern "C" int df_attention_paged4_bf16(const void* q, long long ld_q, const void* cache, const int* page_table_dev,
                                        const int* seq_lens_dev, const int* row_starts_dev, const int* new_lens_dev, void* out,
                                        long long ld_out, int rows, int requests, int max_pages, int num_pages, int page_size,
                                        int q_heads, int kv_heads, int head_dim, int max_new, float scale, void* workspace,
                                        size_t workspace_bytes, int max_ctas, df_status_t* dev_status, void* stream) {
  using namespace df;
  using namespace df::paged;
  if (q == nullptr || cache == nullptr || page_table_dev == nullptr || seq_lens_dev == nullptr || out == nullptr || workspace == nullptr ||
      dev_status == nullptr)
    return fail(DF_EINVAL, "NULL pointer argument");
  if ((row_starts_dev == nullptr) != (new_lens_dev == nullptr)) return fail(DF_EINVAL, "row_starts and new_lens come together");
  if (new_lens_dev == nullptr && (max_new != 1 || rows < requests))
    return fail(DF_EINVAL, "without new_lens every request has one row: max_new must be 1 and rows at least requests");
  if (head_dim != HEAD_DIM) return fail(DF_EUNSUPPORTED, "head_dim must be %d (got %d)", HEAD_DIM, head_dim);
  if (rows <= 0 || requests <= 0 || max_pages <= 0 || num_pages <= 0 || max_new <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0)
    return fail(DF_EINVAL, "rows, requests, max_pages, num_pages, max_new and the head counts must be positive, q_heads a multiple of kv_heads");
  if (page_size <= 0 || page_size % GRANULE != 0) return fail(DF_EINVAL, "page_size must be a positive multiple of %d (got %d)", GRANULE, page_size);
  const long long columns = static_cast<long long>(max_new) * (q_heads / kv_heads);
  const int cols = attn_columns(columns);
  if (static_cast<long long>(max_pages) * page_size > 0x7fffffffLL)
    return fail(DF_EUNSUPPORTED, "max_pages * page_size must stay below 2^31");
  // the list of tiles is numbered with 32 bits
  const double most = static_cast<double>(requests) * (static_cast<double>(max_pages) * page_size / TILE + 1 + SEGMENT_COST) * kv_heads *
                      static_cast<double>((columns + cols - 1) / cols);
  if (columns >= MAX_COLUMNS || kv_heads >= MAX_COLUMNS || most >= 2147483648.0)
    return fail(DF_EUNSUPPORTED, "requests * (max_pages * page_size / %d + %u) * kv_heads * ceil(max_new * group / %d) must stay below 2^31", TILE, SEGMENT_COST + 1, cols);
  if (static_cast<long long>(requests) * max_new > 0x7fffffffLL / q_heads / 4)
    return fail(DF_EUNSUPPORTED, "requests * max_new * q_heads must stay below 2^29");
  if (ld_q < static_cast<long long>(q_heads) * HEAD_DIM || ld_out < static_cast<long long>(q_heads) * HEAD_DIM || (ld_q % 8) != 0 || (ld_out % 8) != 0)
    return fail(DF_EINVAL, "row strides must cover the heads and be multiples of 8 elements");
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15u) != 0)
    return fail(DF_EINVAL, "q, the cache, out and the workspace must be 16-byte aligned");
  if (!(scale > 0.0f)) return fail(DF_EINVAL, "scale must be positive");
  const size_t need = df_attention_paged4_workspace_bytes(requests, q_heads, kv_heads, max_new);
  if (workspace_bytes < need) return fail(DF_EINVAL, "workspace of %zu bytes is too small (need %zu)", workspace_bytes, need);
  const int sms = df_sm_count();
  if (sms <= 0) return fail(DF_ECUDA, "no CUDA device");
  int grid = sms < ATTN_MAX_CTAS ? sms : ATTN_MAX_CTAS;
  if (max_ctas > 0 && max_ctas < grid) grid = max_ctas;
  AttnParams p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.cache = static_cast<const uint8_t*>(cache);
  p.table = page_table_dev;
  p.seq_lens = seq_lens_dev;
  p.row_starts = row_starts_dev;
  p.new_lens = new_lens_dev;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.arrived = static_cast<int*>(workspace);
  p.prefix = reinterpret_cast<uint2*>(static_cast<uint8_t*>(workspace) + attn_counter_bytes());
  p.partial = reinterpret_cast<float*>(p.prefix + (requests + 1) / 2 * 2);
  p.heads = p.partial + static_cast<size_t>(ATTN_MAX_CTAS) * 2 * cols * PARTIAL_FLOATS;
  p.ld_q = ld_q;
  p.ld_out = ld_out;
  p.rows = rows;
  p.requests = requests;
  p.max_pages = max_pages;
  p.num_pages = num_pages;
  p.page_granules = page_size / GRANULE;
  p.q_heads = q_heads;
  p.kv_heads = kv_heads;
  p.group = q_heads / kv_heads;
  p.max_new = max_new;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.inv_group = 1.0f / static_cast<float>(p.group);
  p.timeout_ns = timeout_ns();
  p.status = reinterpret_cast<Status*>(dev_status);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return cols == 8 ? launch_attention<1, attn_warps(8), 2>(p, grid, s) : launch_attention<2, attn_warps(16), 2>(p, grid, s);
}
