// The softmax weights of cached keys, gathered for the block-scaled paged int8 cache (block8.hpp): what a
// cache that is kept within a budget decides by. No counterpart in the reference.
//
// Rows are quantised and scores taken as by the attention where it gives the logarithms of the rows' sums
// (attn_block8.hip; rotations in 64 bits, so that both find the same codes); with a row's, a key's weight in it is
// known without a second look at the keys:
//   w_j <- (j < len - n ? decay * w_j : 0) + sum over the n new rows i that see j, over the group's
//          heads, of 2^(s_ij - lse_i log2 e)
// for each KV head. Bound by the bytes of K for few rows, by the exponentials (VALU, a quarter of the rate of other
// instructions) for many. A call among others (us): 32 x 1 token behind 1024 to 8191, 32 / 8 heads, D = 128, 35 (K's
// 122 MB take 24 at the rate of a copy); 6 x 20 to 33 tokens behind up to 3001 with a window, D = 64, 16, the host's
// call; 2048 tokens behind 2048 keys, 32 / 8 heads, 65 (51 G operations, 24 at the rate of a large int8 product; 201
// million exponentials, 23 at theirs; beside each a conversion, a product and a sum). Kernels in a trace of 30 calls, where
// clocks are lower and launches apart (calls 40, 42 and 77): rows 4.0, keys 28; 3.0 and 7.5; 15, 58, join 5.
#include <algorithm>
#include <climits>

#include "attn_common.hpp"
#include "block8.hpp"
#include "rowquant.hpp"

namespace sl8 {
namespace {

constexpr int AW_THREADS = 256, AW_KEYS = 64;  // keys of an item

struct WeightArgs {
  Block8Seqs s;
  const uint16_t* q;
  const float* lse;
  const int8_t* k;
  const float* ks;
  float* w;
  int64_t wb, wh;  // strides of sequence and head
  int Hq, Hkv, G;
  float q_mul, decay;
  int window;
  bool rotate;
  int8_t* codes;  // [Hkv][D / 64][T * G][64]: a load's 16 rows next to each other (below)
  float2* rows;   // [Hkv][T * G]: scale * q_mul, lse * log2 e
  int parts;      // of an item's rows
  int items;      // at most
  float* part;    // [parts][items][64], parts > 1
};

// The rows as codes, KV head by KV head.
template <int DT, int D>
__global__ void __launch_bounds__(AW_THREADS) weights_rows_kernel(const WeightArgs p) {
  constexpr int LPR = row_lanes(D), RPB = AW_THREADS / LPR;
  const int lane = threadIdx.x % LPR;
  const uint32_t n = (uint32_t)p.s.T * p.Hq, i = blockIdx.x * RPB + threadIdx.x / LPR;  // below 2^30
  const uint32_t row = min(i, n - 1);  // (whole waves: rows past the last repeat it)
  const uint32_t t = row / (uint32_t)p.Hq, h = row - t * p.Hq, kvh = h / (uint32_t)p.G;
  float f[8];
  VecIO<DT>::unpack(reinterpret_cast<const uint4*>(p.q + (int64_t)row * D)[lane], f);
  float safe;
  const uint2 c = row_codes_wide<D>(f, lane, p.rotate, safe);
  if (i >= n) return;
  const int64_t R = p.s.T * p.G, at = (int64_t)t * p.G + h - kvh * p.G, to = kvh * R + at;
  *reinterpret_cast<uint2*>(p.codes + kvh * R * D + ((lane >> 3) * R + at) * 64 + 8 * (lane & 7)) = c;
  if (lane == 0) {
    const float l = p.lse[row];
    // (a row that sees nothing: no weights)
    p.rows[to] = make_float2(safe * p.q_mul, l == -INFINITY ? INFINITY : l * 1.4426950408889634f);
  }
}

// Loads of what is the same for a whole wave and not written here, beside the vector loads in flight (which are
// waited for in their order).
template <typename T>
__device__ __forceinline__ T uniform(const T* p, int64_t i) {
  return reinterpret_cast<const __attribute__((address_space(4))) T*>(reinterpret_cast<uint64_t>(p))[i];
}

// An item: 64 keys of a sequence and KV head, items being the tiles of all sequences in order, a KV head after the
// other.
struct KeyTile {
  int b, kvh, key0, len;  // b < 0: none
  int64_t at[AW_KEYS / 16];  // rows of the cache, by groups of 16 keys; those without a block read the first ones
  float ks[AW_KEYS / 16], off[AW_KEYS / 16];  // and have off -inf
  int64_t row0;
  int n, pos0;
};
// lens: of sequence `lane` of the first 64
__device__ __forceinline__ KeyTile key_tile(const WeightArgs& p, int lane, int lens, int id) {
  KeyTile k;
  k.b = -1;
  const int unit = id / p.Hkv, cap = p.s.maxb * p.s.bs;
  k.kvh = id - unit * p.Hkv;
  int before = 0;
  for (int b0 = 0; b0 < p.s.B; b0 += 64) {
    if (b0) lens = b0 + lane < p.s.B ? p.s.lens[b0 + lane] : 0;
    const int mine = (min(max(lens, 0), cap) + AW_KEYS - 1) / AW_KEYS, sum = before + wave_scan(mine);
    const uint64_t past = __builtin_amdgcn_ballot_w64(sum > unit);
    if (past) {
      const int at = __builtin_ctzll(past);
      k.b = b0 + at;
      k.key0 = (unit - __builtin_amdgcn_readlane(sum - mine, at)) * AW_KEYS;
      const int ctx = __builtin_amdgcn_readlane(lens, at);
      k.len = min(ctx, cap);
      // (no branches between the loads, which wait for each other only as they must)
      const int64_t c0 = p.s.cu ? uniform(p.s.cu, k.b) : k.b, c1 = p.s.cu ? uniform(p.s.cu, k.b + 1) : k.b + 1;
      int blk[AW_KEYS / 16], off[AW_KEYS / 16];
#pragma unroll
      for (int g = 0; g < AW_KEYS / 16; ++g) {
        const int key = k.key0 + 16 * g, j = key / p.s.bs;
        off[g] = key - j * p.s.bs;
        blk[g] = uniform(p.s.table, (int64_t)k.b * p.s.maxb + min(j, p.s.maxb - 1));
      }
      const int64_t r0 = min(max(c0, (int64_t)0), p.s.T), r1 = min(max(c1, (int64_t)0), p.s.T);
      k.row0 = r0;
      k.n = (int)max(r1 - r0, (int64_t)0);
      k.pos0 = (int)min(max((int64_t)ctx - k.n, (int64_t)-(1 << 28)), (int64_t)1 << 30);
#pragma unroll
      for (int g = 0; g < AW_KEYS / 16; ++g) {
        const bool in = k.key0 + 16 * g < k.len && blk[g] >= 0 && blk[g] < p.s.num_blocks;
        const int64_t bh = in ? (int64_t)blk[g] * p.Hkv + k.kvh : 0;
        k.at[g] = in ? bh * p.s.bs + off[g] : 0;
        const float ks = uniform(p.ks, bh);
        k.ks[g] = in ? ks : 0.f;  // (the first block's may be anything)
        k.off[g] = in ? 0.f : -INFINITY;
      }
      break;
    }
    before = __builtin_amdgcn_readlane(sum, 63);
  }
  return k;
}

// The rows that see any of an item's keys, (token, head of the group) in order, and whether there is nothing to do.
struct Rows {
  int r0, r1;
  bool stay;  // behind every window, and no fading
};
__device__ __forceinline__ Rows rows_of(const WeightArgs& p, const KeyTile& it) {
  const int64_t t0 = max(0, it.key0 - it.pos0);
  const int64_t t1 = p.window < 0 ? it.n : min((int64_t)it.n, (int64_t)it.key0 + AW_KEYS - 1 + p.window - it.pos0);
  const int r0 = (int)min(t0, (int64_t)it.n) * p.G, r1 = (int)max(t1, (int64_t)0) * p.G;
  return {r0, r1, r0 >= r1 && p.decay == 1.f && min(it.key0 + AW_KEYS, it.len) <= it.pos0};
}
// The key that a lane puts out: lane (g4, col) key 16 (col / 4) + 4 g4 + col % 4.
__device__ __forceinline__ int key_of(const KeyTile& it, int lane) {
  return it.key0 + 16 * ((lane & 15) >> 2) + 4 * (lane >> 4) + (lane & 3);
}
__device__ __forceinline__ void put(const WeightArgs& p, const KeyTile& it, int key, float was, float sum) {
  if (key < it.len) p.w[it.b * p.wb + it.kvh * p.wh + key] = key < it.pos0 ? fmaf(was, p.decay, sum) : sum;
}

// 64 keys an item. WAVES 1: each wave for itself, its keys' loads being what counts; else the waves of a
// workgroup share the rows (of part blockIdx.y of them) and their sums meet in LDS. Keys are A operands in registers
// (v_mfma_i32_16x16x64_i8), 16 rows at a time the B operands; lane (g4, col) then has keys 16 g + 4 g4 + i for row col.
// (Two waves a SIMD as the least: with one the products go to accumulation registers and are copied back. Rows of
// codes lie 64 bytes at a time, so that a load's 16 are whole lines: in rows of D bytes, two loads to each line, waves
// waited for them in 55 % of their cycles, 19 % now, and 8000 tokens behind 100 keys took 332 us, 280 now.)
template <int D, int WAVES>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES, 2) weights_kernel(const WeightArgs p) {
  constexpr int KS = D / 64, KG = AW_KEYS / 16;
  __shared__ float sum_s[WAVES == 1 ? 1 : WAVES][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g4 = lane >> 4;
  const int lens = lane < p.s.B ? p.s.lens[lane] : 0;
  // every other part begins from the end: the tiles of a causal prompt are seen by fewer rows the later they are
  for (int x = blockIdx.y & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x;; x += gridDim.x) {
    // WAVES 1: four tiles of a head next to each other (32 x 1 token 34.5 us, 35 where they are of four heads)
    const int id = WAVES == 1 ? (x / p.Hkv * 4 + wave) * p.Hkv + x % p.Hkv : x;
    const KeyTile it = key_tile(p, lane, lens, id);
    if (it.b < 0) return;
    const Rows all = rows_of(p, it);
    if (all.stay) continue;
    int r0 = all.r0, r1 = all.r1;
    if (WAVES > 1 && p.parts > 1) {
      const int per = ((r1 - r0 + 15) / 16 + p.parts - 1) / p.parts * 16;
      r0 = min(r0 + (int)blockIdx.y * per, r1);
      r1 = min(r0 + per, r1);
    }
    const int key0 = it.key0, pos0 = it.pos0;
    v4i ka[KG][KS];
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      const int8_t* from = p.k + (it.at[g] + col) * D + 16 * g4;
#pragma unroll
      for (int s = 0; s < KS; ++s) ka[g][s] = *reinterpret_cast<const v4i*>(from + 64 * s);
    }
    const int key = key_of(it, lane);
    const float was = p.w[it.b * p.wb + it.kvh * p.wh + min(key, it.len - 1)];
    const int64_t R = p.s.T * p.G;
    const int8_t* codes = p.codes + it.kvh * R * D + it.row0 * p.G * 64;
    const float2* rows = p.rows + ((int64_t)it.kvh * p.s.T + it.row0) * p.G;
    // rows from `seen` on see all of the keys, up to `until` (row units; a window's side)
    const int seen = (int)min((int64_t)max(key0 + AW_KEYS - 1 - pos0, 0) * p.G, (int64_t)INT_MAX);
    const int until = p.window < 0 ? INT_MAX
                                   : (int)min(max(((int64_t)key0 - pos0 + p.window) * p.G, (int64_t)0), (int64_t)INT_MAX);
    float acc[KG][4] = {};
    const int rw = r0 + (WAVES == 1 ? 0 : 16 * wave);
    v4i q0[KS], q1[KS];
    float2 y0, y1;
    auto load = [&](int r, v4i (&q)[KS], float2& s) __attribute__((always_inline)) {
      r = min(r, r1 - 1);  // (past the last: as the last)
      const uint32_t row = min(col, r1 - 1 - r);
#pragma unroll
      for (int i = 0; i < KS; ++i) q[i] = *reinterpret_cast<const v4i*>(codes + (i * R + r) * 64 + (64 * row + 16 * g4));
      s = (rows + r)[row];
    };
    auto pass = [&](int r, const v4i (&q)[KS], float2 y, v4i (&next)[KS], float2& yn) __attribute__((always_inline)) {
      load(r + 16 * WAVES, next, yn);
      v4i sc[KG];
#pragma unroll
      for (int g = 0; g < KG; ++g) {
        sc[g] = v4i{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) sc[g] = __builtin_amdgcn_mfma_i32_16x16x64_i8(ka[g][s], q[s], sc[g], 0, 0, 0);
      }
      float e[KG][4];
#pragma unroll
      for (int g = 0; g < KG; ++g) {
        const float a = y.x * it.ks[g], c = it.off[g] - y.y;
#pragma unroll
        for (int i = 0; i < 4; ++i) e[g][i] = __builtin_amdgcn_exp2f(fmaf((float)sc[g][i], a, c));
      }
      if (!(r >= seen && r + 15 < until && r + 16 <= r1)) {  // each row its own
        // (places counted from the lane's first key)
        const int pos = pos0 + (r + col) / p.G - key0 - 4 * g4, lim = r + col < r1 ? pos + 1 : 0;
        const int low = p.window >= 0 ? pos - p.window + 1 : 0;
#pragma unroll
        for (int g = 0; g < KG; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * g + i >= lim || 16 * g + i < low) e[g][i] = 0.f;
      }
#pragma unroll
      for (int g = 0; g < KG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[g][i] += e[g][i];
    };
    if (rw < r1) load(rw, q0, y0);
    if constexpr (WAVES > 1) {
      for (int r = rw; r < r1; r += 32 * WAVES) {
        pass(r, q0, y0, q1, y1);
        if (r + 16 * WAVES < r1) pass(r + 16 * WAVES, q1, y1, q0, y0);
      }
    } else {  // (one pass for the most part: fewer registers, a wave a SIMD more at D = 128)
      for (int r = rw; r < r1; r += 16) {
        pass(r, q0, y0, q1, y1);
#pragma unroll
        for (int i = 0; i < KS; ++i) q0[i] = q1[i];
        y0 = y1;
      }
    }
    // over the 16 rows of a lane group; lane (g4, col) keeps key 16 (col / 4) + 4 g4 + col % 4
    float sum = 0.f;
#pragma unroll
    for (int g = 0; g < KG; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v = acc[g][i];
        auto add = [&](auto ctrl) __attribute__((always_inline)) {
          v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xF, 0xF, false));
        };
        using std::integral_constant;
        add(integral_constant<int, 0xB1>{});   // quad_perm 1,0,3,2
        add(integral_constant<int, 0x4E>{});   // quad_perm 2,3,0,1
        add(integral_constant<int, 0x141>{});  // row_half_mirror
        add(integral_constant<int, 0x140>{});  // row_mirror
        if (col == 4 * g + i) sum = v;
      }
    if constexpr (WAVES > 1) {
      sum_s[wave][lane] = sum;
      __syncthreads();
      if (wave == 0) {
        sum = 0.f;
#pragma unroll
        for (int x = 0; x < WAVES; ++x) sum += sum_s[x][lane];
        if (p.parts > 1) p.part[((int64_t)blockIdx.y * p.items + id) * AW_KEYS + lane] = sum;
        else put(p, it, key, was, sum);
      }
      __syncthreads();  // (the next item's sums go to the same place)
    } else {
      put(p, it, key, was, sum);
    }
  }
}

// The parts of the rows added up, in their order: a wave an item.
__global__ void __launch_bounds__(256) weights_join_kernel(const WeightArgs p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lens = lane < p.s.B ? p.s.lens[lane] : 0;
  const KeyTile it = key_tile(p, lane, lens, blockIdx.x * 4 + wave);
  if (it.b < 0 || rows_of(p, it).stay) return;
  const int key = key_of(it, lane);
  const float was = p.w[it.b * p.wb + it.kvh * p.wh + min(key, it.len - 1)];
  float sum = 0.f;
#pragma unroll 8
  for (int s = 0; s < p.parts; ++s) sum += p.part[((int64_t)s * p.items + blockIdx.x * 4 + wave) * AW_KEYS + lane];
  put(p, it, key, was, sum);
}

// How a call runs: rows of a sequence and KV head on average, items at most, and in how many parts the rows of an
// item go to workgroups of their own: where items are few, so that there are two for each CU, and four where new rows
// are a good part of the context (a causal prompt's last keys are seen by few of its rows, so items differ); parts
// large enough to pay for the join. Whole and in parts (us): 2000 rows behind 100 keys, 8 heads to a KV head, D = 256,
// 134 and 35; 4000 behind 100, 8 / 2 heads, D = 128, 134 and 51; 2048 behind 2048, 32 / 8 heads, 101 and 92, later 75
// (6 parts for 2: 87); 700 behind 30000, 8 / 1 heads, 60 whole, 84 in two.
// A wave an item for up to 32 rows, else four: one row, 32 sequences 32 and 96; 16 tokens of 4 heads, D = 64, 18.8 and
// 20.3; 300 of 4 heads, D = 128, 47 and 24. (By the batch's average: lengths are on the device.)
struct WeightPlan {
  int64_t rows, items, parts;
  size_t rows_at, part_at, bytes;
};
constexpr int AW_WAVES = 4;
// Workgroups of the pass over the rows, and whether a launch (below 2^32 threads) holds them.
int64_t rows_wgs(int64_t rows, int64_t D) {
  const int64_t per = AW_THREADS / row_lanes((int)D);
  return (rows + per - 1) / per;
}
bool rows_fit(int64_t rows, int64_t D) { return rows < (1LL << 30) && rows_wgs(rows, D) < (1LL << 32) / AW_THREADS; }
WeightPlan weights_plan(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t cap) {
  WeightPlan a{};
  a.rows = T * (Hq / Hkv) / B;
  a.items = B * Hkv * ((cap + AW_KEYS - 1) / AW_KEYS);
  a.parts = 1;
  if (a.rows > 32 && a.items > 0) {
    const bool uneven = T / B * 4 >= cap;
    const int64_t want = (int64_t)cu_count() * (uneven ? 4 : 2) / a.items;
    a.parts = std::max<int64_t>(1, std::min<int64_t>({want, a.rows / (uneven ? 1024 : 512), 64}));
  }
  a.rows_at = (size_t)(T * Hq) * D;
  a.part_at = a.rows_at + (size_t)(T * Hq) * sizeof(float2);
  a.bytes = a.part_at + (a.parts > 1 ? (size_t)(a.parts * a.items) * AW_KEYS * sizeof(float) : 0);
  return a;
}

}  // namespace
}  // namespace sl8

using namespace sl8;

extern "C" size_t sl8_attn_weights_block8_workspace(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                                                    int64_t max_context_len) {
  if (T <= 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || T >= (1LL << 28) || B >= (1 << 24) || Hq >= (1 << 16)) return 0;
  if ((D != 64 && D != 128 && D != 256) || Hq % Hkv || max_context_len < 0 || max_context_len >= (1LL << 30)) return 0;
  if (B * Hkv * (max_context_len / AW_KEYS + 1) >= (1LL << 30) || !rows_fit(T * Hq, D)) return 0;
  return weights_plan(T, B, Hq, Hkv, D, max_context_len).bytes;
}

extern "C" int sl8_attn_weights_block8(const void* q, int dtype, int rotate, float q_scale_mul, const float* lse,
                                       const int8_t* k_cache, const float* k_scale, const int32_t* cu_lens,
                                       const int32_t* context_lens, const int32_t* block_table, float* weights,
                                       int64_t weights_stride_b, int64_t weights_stride_h, float decay, int64_t T,
                                       int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t num_blocks,
                                       int64_t block_size, int64_t max_blocks_per_seq, int64_t window_left,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  const char* tag = "attn_weights_block8";
  SL8_CHECK_ARG(dtype == SL8_DTYPE_F16 || dtype == SL8_DTYPE_BF16, "fni8 %s: q must be float16 or bfloat16", tag);
  SL8_CHECK_ARG(T >= 0 && T < (1LL << 28) && B >= 0 && B < (1 << 24) && Hq >= 0 && Hq < (1 << 16) &&
                    num_blocks >= 0 && num_blocks < (1LL << 31) && max_blocks_per_seq >= 0 &&
                    max_blocks_per_seq < (1LL << 31) && block_size >= 0 && block_size < (1 << 16),
                "fni8 %s: shape too large", tag);
  WeightArgs p{};
  p.s = Block8Seqs{cu_lens, context_lens, block_table, T, (int)B, (int)max_blocks_per_seq, (int)num_blocks,
                   (int)block_size};
  if (const int rc = block8_check(tag, p.s, Hkv, D)) return rc;
  SL8_CHECK_ARG(Hq > 0 && Hq % Hkv == 0, "fni8 %s: H_q must be divisible by H_kv (GQA)", tag);
  SL8_CHECK_ARG(rows_fit(T * Hq, D), "fni8 %s: shape too large", tag);
  if (B == 0 || max_blocks_per_seq == 0) return SL8_OK;
  SL8_CHECK_ARG(num_blocks > 0, "fni8 %s: the cache has no blocks", tag);
  SL8_CHECK_ARG(context_lens && block_table && weights && k_cache && k_scale &&
                    (T == 0 || (q && lse)),
                "fni8 %s: null pointer", tag);
  SL8_CHECK_ARG(aligned(q, 16) && aligned(k_cache, 16), "fni8 %s: q/k_cache must be 16-byte aligned", tag);
  const int64_t cap = max_blocks_per_seq * block_size;
  SL8_CHECK_ARG(B * Hkv * (cap / AW_KEYS + 1) < (1LL << 30), "fni8 %s: shape too large", tag);
  const WeightPlan plan = weights_plan(T, B, Hq, Hkv, D, cap);
  SL8_CHECK_ARG(T == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= plan.bytes),
                "fni8 %s: workspace needs %zu bytes", tag, plan.bytes);
  p.q = static_cast<const uint16_t*>(q);
  p.lse = lse;
  p.k = k_cache; p.ks = k_scale;
  p.w = weights; p.wb = weights_stride_b; p.wh = weights_stride_h;
  p.Hq = (int)Hq; p.Hkv = (int)Hkv; p.G = (int)(Hq / Hkv);
  p.q_mul = q_scale_mul;
  p.decay = decay;
  p.rotate = rotate != 0;
  p.window = window_left < 0 ? -1 : (int)(window_left < (1 << 30) ? window_left : (1 << 30));
  p.codes = static_cast<int8_t*>(workspace);
  p.rows = reinterpret_cast<float2*>(p.codes + plan.rows_at);
  p.part = reinterpret_cast<float*>(p.codes + plan.part_at);
  p.parts = (int)plan.parts;
  p.items = (int)plan.items;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  auto by_d = [&](auto d) {
    constexpr int DD = decltype(d)::value;
    const unsigned pre = (unsigned)rows_wgs(T * Hq, DD);
    if (T) {
      if (dtype == SL8_DTYPE_F16) weights_rows_kernel<SL8_DTYPE_F16, DD><<<pre, AW_THREADS, 0, st>>>(p);
      else weights_rows_kernel<SL8_DTYPE_BF16, DD><<<pre, AW_THREADS, 0, st>>>(p);
    }
    const int64_t cus = cu_count();
    if (plan.rows <= 32) {
      const int64_t groups = (B * ((cap + AW_KEYS - 1) / AW_KEYS) + 3) / 4 * Hkv;
      weights_kernel<DD, 1><<<(unsigned)std::min(groups, cus * 8), 256, 0, st>>>(p);
    } else {
      const dim3 grid((unsigned)std::min(plan.items, cus * 12), (unsigned)plan.parts);
      weights_kernel<DD, AW_WAVES><<<grid, 64 * AW_WAVES, 0, st>>>(p);
      if (plan.parts > 1) weights_join_kernel<<<(unsigned)((plan.items + 3) / 4), 256, 0, st>>>(p);
    }
  };
  if (D == 64) by_d(std::integral_constant<int, 64>{});
  else if (D == 128) by_d(std::integral_constant<int, 128>{});
  else by_d(std::integral_constant<int, 256>{});
  SL8_CHECK_LAUNCH(tag);
  return SL8_OK;
}
