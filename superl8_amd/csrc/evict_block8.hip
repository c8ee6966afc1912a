// Eviction from the block-scaled paged int8 cache (block8.hpp) by the keys' gathered weights. No
// counterpart in the reference.
//
// Of each sequence and KV head m = min(len, budget) tokens stay: the first `sinks`, the last `recent`, and
// of those between the ones of the largest weights, ties to the lowest index. They keep their order and move
// into other blocks, those of a second table, which the call writes and never reads; so blocks that
// sequences share are only read. A block takes
//   s' = max(scales of the blocks that its rows come from, 2^-60), codes c' = rint(c * (s / s')),
// so rows that stay together, or come from blocks of one scale, are copied as they are.
//
// Bound by the counting, which has a workgroup for each sequence and head, and by the kept rows' bytes, K and V, in
// and out. Kernels (us): 4 sequences of 733 to 1100 tokens to 1024, 8 heads, D = 128, select 7.7, move 7.5 (the 17 MB
// of rows come from and go to caches); 8 of 21845 to 32768 to 4096 select 26, move 31 (134 MB, 26 at a copy's rate).
#include <algorithm>

#include "block8.hpp"
#include "rowquant.hpp"

namespace sl8 {
namespace {

constexpr int EV_THREADS = 1024, EV_WAVES = EV_THREADS / 64;

struct EvictArgs {
  Block8Seqs s;  // of the tokens as they are
  int8_t *k, *v;
  float *ks, *vs;
  float* w;
  int64_t wb, wh;
  const int32_t* to;  // [B][to_maxb]
  int to_maxb;
  int32_t* kept;  // [B][Hkv][budget]
  int32_t* lens;  // [B]
  int Hkv, budget, sinks, recent;

  __device__ __forceinline__ int len(int b) const { return min(max(s.lens[b], 0), s.maxb * s.bs); }
};

// Weights in the order of unsigned numbers (-0 as 0).
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float weight_of(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u); }

// What the waves of a workgroup add up, in their order: (sum of the waves before, of all).
__device__ __forceinline__ int2 over_waves(int mine, int wave, int* sums) {
  if ((threadIdx.x & 63) == 63) sums[wave] = mine;
  __syncthreads();
  int2 r = make_int2(0, 0);
#pragma unroll
  for (int x = 0; x < EV_WAVES; ++x) {
    if (x < wave) r.x += sums[x];
    r.y += sums[x];
  }
  return r;
}

// A workgroup for each sequence and KV head. The least weight that stays is found by counting: 2048 bins over the
// range that the weights take (by their bits as whole numbers: a bin's count rarely meets another's atomics there,
// as the highest byte's would), then over the bin that holds it, three times at most. Which stay then follows in
// order from the counts of each 64. VPT weights a thread are kept in registers; 0: longer contexts are read again
// for each count (32768 tokens so: 67 us for 27).
template <int VPT>
__global__ void __launch_bounds__(EV_THREADS) evict_select_kernel(const EvictArgs p) {
  constexpr int BINS = 2048, ROWS = VPT ? VPT : 1;
  __shared__ int hist[BINS];
  __shared__ int sums_a[EV_WAVES], sums_b[EV_WAVES];
  __shared__ uint32_t ends_s[2][EV_WAVES];
  __shared__ int found_s[2];
  __shared__ int wave_s[ROWS][EV_WAVES], eq_s[ROWS][EV_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x - b * p.Hkv;
  const int len = p.len(b), m = min(len, p.budget);
  float* w = p.w + b * p.wb + h * p.wh;
  int32_t* kept = p.kept + (int64_t)blockIdx.x * p.budget;
  if (h == 0 && tid == 0) p.lens[b] = m;
  for (int i = m + tid; i < p.budget; i += EV_THREADS) kept[i] = -1;
  if (m == len) {
    for (int i = tid; i < m; i += EV_THREADS) kept[i] = i;
    return;
  }
  // between the first and the last ones the weights decide (sinks + recent <= budget < len)
  const int first = p.sinks, last = len - p.recent;
  uint32_t u[ROWS];
  if constexpr (VPT > 0) {
    float x[ROWS];
#pragma unroll
    for (int c = 0; c < VPT; ++c) x[c] = w[min(c * EV_THREADS + tid, len - 1)];
#pragma unroll
    for (int c = 0; c < VPT; ++c) u[c] = order_of(x[c]);
  }
  auto each = [&](auto f) __attribute__((always_inline)) {  // f(weight) of those between
    if constexpr (VPT > 0) {
#pragma unroll
      for (int c = 0; c < VPT; ++c) {
        const int i = c * EV_THREADS + tid;
        if (i >= first && i < last) f(u[c]);
      }
    } else {
      for (int i = first + tid; i < last; i += EV_THREADS) f(order_of(w[i]));
    }
  };
  int want = m - p.sinks - p.recent;
  uint32_t least = 0xFFFFFFFFu;
  int equal = 0;  // how many of the least stay
  if (want > 0) {
    uint32_t lo = 0xFFFFFFFFu, hi = 0;
    each([&](uint32_t x) {
      lo = min(lo, x);
      hi = max(hi, x);
    });
    lo = ~lane_group_reduce<64>(~lo, [](uint32_t a, uint32_t c) { return a > c ? a : c; });
    hi = lane_group_reduce<64>(hi, [](uint32_t a, uint32_t c) { return a > c ? a : c; });
    if (lane == 0) {
      ends_s[0][wave] = lo;
      ends_s[1][wave] = hi;
    }
    for (int i = tid; i < BINS; i += EV_THREADS) hist[i] = 0;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < EV_WAVES; ++x) {
      lo = min(lo, ends_s[0][x]);
      hi = max(hi, ends_s[1][x]);
    }
    uint32_t base = lo, span = hi - lo;  // the one looked for is in [base, base + span]
    for (;;) {
      const int bits = 32 - __clz((int)span);  // (of 0: 0)
      const int shift = max(bits - 11, 0);
      each([&](uint32_t x) {
        const uint32_t d = x - base;
        if (x >= base && d <= span) atomicAdd(&hist[d >> shift], 1);
      });
      __syncthreads();
      // bins from the highest, two a thread
      const int b0 = BINS - 1 - 2 * tid;
      const int h0 = hist[b0], h1 = hist[b0 - 1];
      const int upto = wave_scan(h0 + h1);
      const int2 before = over_waves(upto, wave, sums_a);
      const int above = before.x + upto - h0 - h1;
      if (above < want && want <= above + h0 + h1) {  // (one thread)
        const bool second = want > above + h0;
        found_s[0] = second ? b0 - 1 : b0;
        found_s[1] = want - above - (second ? h0 : 0);
      }
      hist[b0] = 0;
      hist[b0 - 1] = 0;
      __syncthreads();
      base += (uint32_t)found_s[0] << shift;
      want = found_s[1];
      if (shift == 0) break;
      span = min(span, (1u << shift) - 1);
      __syncthreads();
    }
    least = base;
    equal = want;
  }
  if constexpr (VPT > 0) {
    // counts of each 64, then where their kept ones go
    uint64_t eqs[ROWS], sures[ROWS];
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
      const int i = c * EV_THREADS + tid;
      const bool between = i >= first && i < last;
      eqs[c] = __ballot(between && equal > 0 && u[c] == least);
      sures[c] = __ballot(i < len && (!between || u[c] > least));
      if (lane == 0) {
        eq_s[c][wave] = __popcll(eqs[c]);
        wave_s[c][wave] = __popcll(sures[c]);
      }
    }
    __syncthreads();
    const int e = tid < VPT * EV_WAVES ? (&eq_s[0][0])[tid] : 0, s = tid < VPT * EV_WAVES ? (&wave_s[0][0])[tid] : 0;
    const int es = wave_scan(e);
    const int eq0 = over_waves(es, wave, sums_a).x + es - e;  // equal ones in front
    const int k = s + min(eq0 + e, equal) - min(eq0, equal);
    const int ks = wave_scan(k);
    const int at0 = over_waves(ks, wave, sums_b).x + ks - k;
    if (tid < VPT * EV_WAVES) {
      (&eq_s[0][0])[tid] = eq0;
      (&wave_s[0][0])[tid] = at0;
    }
    __syncthreads();
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
      const int i = c * EV_THREADS + tid;
      const int base_eq = eq_s[c][wave], rank = base_eq + __popcll(eqs[c] & below);
      const bool sure = sures[c] >> lane & 1, eq = eqs[c] >> lane & 1;
      if (sure || (eq && rank < equal)) {
        const int at = wave_s[c][wave] + __popcll(sures[c] & below) + min(rank, equal) - min(base_eq, equal);
        kept[at] = i;
        w[at] = weight_of(u[c]);
      }
    }
    return;
  }
  // in order, a weight a thread: how many equal ones and how many kept ones stand in front
  int equals = 0, keeps = 0;
  for (int from = 0; from < len; from += EV_THREADS) {
    const int i = from + tid;
    const float x = i < len ? w[i] : 0.f;
    const bool between = i >= first && i < last;
    const uint32_t v = order_of(x);
    const bool eq = between && equal > 0 && v == least;
    const bool sure = i < len && (!between || v > least);
    const uint64_t eqs = __ballot(eq), sures = __ballot(sure), below = (1ull << lane) - 1;
    const int2 e = over_waves(__popcll(eqs), wave, sums_a);  // (behind its barrier all of these weights are read)
    const int2 s = over_waves(__popcll(sures), wave, sums_b);
    const int rank = equals + e.x + __popcll(eqs & below);
    if (sure || (eq && rank < equal)) {
      const int at = keeps + s.x + __popcll(sures & below) + min(rank, equal) - min(equals, equal);
      kept[at] = i;
      w[at] = x;
    }
    keeps += s.y + min(equals + e.y, equal) - min(equals, equal);
    equals += e.y;
  }
}

// A workgroup for each block that is written and KV head, K and V: a thread has 16 bytes of a row.
template <int D>
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictArgs p, int blocks) {
  constexpr int LPR = D / 16, RPB = 256 / LPR;
  __shared__ float ks_s[BLK8_MAX], vs_s[BLK8_MAX];
  __shared__ int64_t at_s[BLK8_MAX];
  const int h = blockIdx.x % p.Hkv, r = blockIdx.x / p.Hkv;
  const int b = r / blocks, blk = r - b * blocks;
  const int bs = p.s.bs;
  const int m = min(p.len(b), p.budget);
  const int cnt = min(m - blk * bs, bs);
  if (cnt <= 0 || blk >= p.to_maxb) return;
  const int id = p.to[(int64_t)b * p.to_maxb + blk];
  if (id < 0 || id >= p.s.num_blocks) return;
  for (int i = threadIdx.x; i < cnt; i += 256) {
    const int src = p.kept[((int64_t)b * p.Hkv + h) * p.budget + blk * bs + i];
    const int page = p.s.block(b, src / bs);
    const int64_t bh = (int64_t)page * p.Hkv + h;
    at_s[i] = page < 0 ? -1 : (bh * bs + src % bs) * D;
    ks_s[i] = page < 0 ? 0.f : p.ks[bh];
    vs_s[i] = page < 0 ? 0.f : p.vs[bh];
  }
  __syncthreads();
  float kn = 0x1p-60f, vn = 0x1p-60f;
  for (int i = threadIdx.x & 63; i < cnt; i += 64) {
    kn = fmaxf(kn, ks_s[i]);
    vn = fmaxf(vn, vs_s[i]);
  }
  kn = wave_max(kn);
  vn = wave_max(vn);
  const int64_t bh = (int64_t)id * p.Hkv + h;
  if (threadIdx.x == 0) {
    p.ks[bh] = kn;
    p.vs[bh] = vn;
  }
  const int lane = threadIdx.x % LPR;
  for (int i = threadIdx.x / LPR; i < cnt; i += RPB) {
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int8_t* from = side ? p.v : p.k;
      const float was = side ? vs_s[i] : ks_s[i], now = side ? vn : kn;
      uint4 c = make_uint4(0, 0, 0, 0);
      if (at_s[i] >= 0) c = *reinterpret_cast<const uint4*>(from + at_s[i] + 16 * lane);
      if (was != now) {
        const float ratio = __fdiv_rn(was, now);
        uint32_t x[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          uint32_t o = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            o |= (uint32_t)(uint8_t)(int8_t)rintf((float)(int8_t)(x[d] >> (8 * e)) * ratio) << (8 * e);
          x[d] = o;
        }
        c = make_uint4(x[0], x[1], x[2], x[3]);
      }
      *reinterpret_cast<uint4*>((side ? p.v : p.k) + (bh * bs + i) * D + 16 * lane) = c;
    }
  }
}

}  // namespace
}  // namespace sl8

using namespace sl8;

extern "C" int sl8_kv_evict_block8(int8_t* k_cache, float* k_scale, int8_t* v_cache, float* v_scale,
                                   const int32_t* context_lens, const int32_t* block_table, float* weights,
                                   int64_t weights_stride_b, int64_t weights_stride_h, const int32_t* new_table,
                                   int32_t* new_lens, int32_t* kept, int64_t B, int64_t Hkv, int64_t D,
                                   int64_t num_blocks, int64_t block_size, int64_t max_blocks_per_seq,
                                   int64_t new_max_blocks, int64_t budget, int64_t sinks, int64_t recent,
                                   void* stream) {
  clear_error();
  const char* tag = "kv_evict_block8";
  SL8_CHECK_ARG(B >= 0 && B < (1 << 24) && num_blocks >= 0 && num_blocks < (1LL << 31) && max_blocks_per_seq >= 0 &&
                    max_blocks_per_seq < (1LL << 31) && block_size >= 0 && block_size < (1 << 16) &&
                    new_max_blocks >= 0 && new_max_blocks < (1LL << 31) && budget < (1LL << 30),
                "fni8 %s: shape too large", tag);
  EvictArgs p{};
  p.s = Block8Seqs{nullptr, context_lens, block_table, B, (int)B, (int)max_blocks_per_seq, (int)num_blocks,
                   (int)block_size};
  if (const int rc = block8_check(tag, p.s, Hkv, D)) return rc;
  SL8_CHECK_ARG(budget >= 1 && sinks >= 0 && recent >= 0 && sinks <= budget && recent <= budget - sinks,
                "fni8 %s: budget must be at least 1 and hold sinks and recent", tag);
  const int64_t most = std::min(budget, max_blocks_per_seq * block_size);  // tokens that a sequence keeps
  const int64_t blocks = (most + block_size - 1) / block_size;
  SL8_CHECK_ARG(new_max_blocks >= blocks, "fni8 %s: new_table must hold the tokens that stay (%lld blocks)", tag,
                (long long)blocks);
  if (B == 0) return SL8_OK;
  SL8_CHECK_ARG(context_lens && new_lens && kept && (max_blocks_per_seq == 0 || (block_table && weights)) &&
                    (blocks == 0 || new_table) && (num_blocks == 0 || (k_cache && k_scale && v_cache && v_scale)),
                "fni8 %s: null pointer", tag);
  SL8_CHECK_ARG(aligned(k_cache, 16) && aligned(v_cache, 16), "fni8 %s: caches must be 16-byte aligned", tag);
  SL8_CHECK_ARG(B * Hkv < (1LL << 32) / EV_THREADS && B * Hkv * blocks < (1LL << 32) / 256,
                "fni8 %s: shape too large", tag);
  // (a sequence's heads are workgroups of their own, and the first one writes its new length)
  SL8_CHECK_ARG(new_lens + B <= context_lens || context_lens + B <= new_lens,
                "fni8 %s: new_lens must not overlap context_lens", tag);
  p.k = k_cache; p.v = v_cache; p.ks = k_scale; p.vs = v_scale;
  p.w = weights; p.wb = weights_stride_b; p.wh = weights_stride_h;
  p.to = new_table;
  p.to_maxb = (int)new_max_blocks;
  p.kept = kept;
  p.lens = new_lens;
  p.Hkv = (int)Hkv; p.budget = (int)budget; p.sinks = (int)sinks; p.recent = (int)recent;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  auto select = [&](auto vpt) {
    evict_select_kernel<decltype(vpt)::value><<<(unsigned)(B * Hkv), EV_THREADS, 0, st>>>(p);
  };
  const int64_t cap = max_blocks_per_seq * block_size;
  if (cap <= 4 * EV_THREADS) select(std::integral_constant<int, 4>{});
  else if (cap <= 16 * EV_THREADS) select(std::integral_constant<int, 16>{});
  else if (cap <= 32 * EV_THREADS) select(std::integral_constant<int, 32>{});
  else select(std::integral_constant<int, 0>{});
  const unsigned grid = (unsigned)(B * Hkv * blocks);
  if (grid && num_blocks) {
    if (D == 64) evict_move_kernel<64><<<grid, 256, 0, st>>>(p, (int)blocks);
    else if (D == 128) evict_move_kernel<128><<<grid, 256, 0, st>>>(p, (int)blocks);
    else evict_move_kernel<256><<<grid, 256, 0, st>>>(p, (int)blocks);
  }
  SL8_CHECK_LAUNCH(tag);
  return SL8_OK;
}
