// Eviction from the block-scaled paged int8 cache (block8.hpp) by the keys' gathered weights. No
// counterpart in the reference.
//
// Of each sequence and KV head m = min(len, budget) tokens stay: the first `sinks`, the last `recent`, and
// of those between the ones of the largest weights, ties to the lowest index. They keep their order and move
// into other blocks, those of a second table, which the call writes and never reads; so blocks that
// sequences share are only read. A block takes
//   s' = max(scales of the blocks that its rows come from, 2^-60), codes c' = rint(c * (s / s')),
// so rows that stay together, or come from blocks of one scale, are copied as they are.
#include <algorithm>

#include "block8.hpp"

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

// A workgroup for each sequence and KV head: the least weight that stays by its bytes, from the highest
// (how many share the bytes found so far and have which next one), then the kept in order.
__global__ void __launch_bounds__(EV_THREADS) evict_select_kernel(const EvictArgs p) {
  __shared__ int hist[256];
  __shared__ int wave_s[2][EV_WAVES][2];
  __shared__ int found_s[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
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
  const int first = p.sinks, last = len - p.recent;  // between them the weights decide (sinks + recent <= budget < len)
  int want = m - p.sinks - p.recent;
  uint32_t least = 0xFFFFFFFFu;
  int equal = 0;  // how many of the least stay
  if (want > 0) {
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = first + tid; i < last; i += EV_THREADS) {
        const uint32_t u = order_of(w[i]);
        if (shift == 24 || u >> (shift + 8) == prefix) atomicAdd(&hist[u >> shift & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int x = 255, left = want;
        while (x > 0 && hist[x] < left) left -= hist[x--];
        found_s[0] = x;
        found_s[1] = left;
      }
      __syncthreads();
      prefix = prefix << 8 | (uint32_t)found_s[0];
      want = found_s[1];
      __syncthreads();
    }
    least = prefix;
    equal = want;
  }
  // in order: how many equal ones and how many kept ones stand in front
  int equals = 0, keeps = 0;
  for (int base = 0, turn = 0; base < len; base += EV_THREADS, turn ^= 1) {
    const int i = base + tid;
    const float x = i < len ? w[i] : 0.f;
    const bool between = i >= first && i < last;
    const uint32_t u = order_of(x);
    const bool eq = between && want > 0 && u == least && i < len;
    const bool sure = i < len && (!between || (u > least));
    const uint64_t eqs = __ballot(eq), sures = __ballot(sure);
    if (lane == 0) {
      wave_s[turn][wave][0] = __popcll(eqs);
      wave_s[turn][wave][1] = __popcll(sures);
    }
    __syncthreads();  // (all of this turn's weights are read)
    const uint64_t below = (1ull << lane) - 1;
    int e0 = equals, s0 = 0, e_all = 0, s_all = 0;
    for (int x2 = 0; x2 < EV_WAVES; ++x2) {
      const int e = wave_s[turn][x2][0], s = wave_s[turn][x2][1];
      if (x2 < wave) { e0 += e; s0 += s; }
      e_all += e;
      s_all += s;
    }
    const int rank = e0 + __popcll(eqs & below);              // equal ones in front
    const int taken = min(rank, equal) - min(equals, equal);  // of them, those of this turn that stay
    const bool keep = sure || (eq && rank < equal);
    if (keep) {
      const int at = keeps + s0 + __popcll(sures & below) + taken;
      kept[at] = i;
      w[at] = x;
    }
    keeps += s_all + min(equals + e_all, equal) - min(equals, equal);
    equals += e_all;
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
  p.k = k_cache; p.v = v_cache; p.ks = k_scale; p.vs = v_scale;
  p.w = weights; p.wb = weights_stride_b; p.wh = weights_stride_h;
  p.to = new_table;
  p.to_maxb = (int)new_max_blocks;
  p.kept = kept;
  p.lens = new_lens;
  p.Hkv = (int)Hkv; p.budget = (int)budget; p.sinks = (int)sinks; p.recent = (int)recent;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  evict_select_kernel<<<(unsigned)(B * Hkv), EV_THREADS, 0, st>>>(p);
  const unsigned grid = (unsigned)(B * Hkv * blocks);
  if (grid && num_blocks) {
    if (D == 64) evict_move_kernel<64><<<grid, 256, 0, st>>>(p, (int)blocks);
    else if (D == 128) evict_move_kernel<128><<<grid, 256, 0, st>>>(p, (int)blocks);
    else evict_move_kernel<256><<<grid, 256, 0, st>>>(p, (int)blocks);
  }
  SL8_CHECK_LAUNCH(tag);
  return SL8_OK;
}
