// The softmax weights of cached keys, gathered for the block-scaled paged int8 cache (block8.hpp): what a
// cache that is kept within a budget decides by. No counterpart in the reference.
//
// Rows are quantised and scores taken as by the attention (attn_block8.hip); with the logarithm of a row's
// sum, which that attention gives, a key's weight in the row is known without a second look at the keys:
//   w_j <- (j < len - n ? decay * w_j : 0) + sum over the n new rows i that see j, over the group's
//          heads, of 2^(s_ij - lse_i log2 e)
// for each KV head. Bound by the bytes of K for few rows, by the exponentials (VALU) for many.
#include <algorithm>

#include "attn_common.hpp"
#include "block8.hpp"
#include "rowquant.hpp"

namespace sl8 {
namespace {

constexpr int AW_THREADS = 256, AW_KEYS = 256;  // keys of a workgroup, 64 a wave

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
  int8_t* codes;  // [Hkv][T * G][D]
  float2* rows;   // [Hkv][T * G]: scale * q_mul, lse * log2 e
};

// The rows as codes, KV head by KV head.
template <int DT, int D>
__global__ void __launch_bounds__(AW_THREADS) weights_rows_kernel(const WeightArgs p) {
  constexpr int LPR = row_lanes(D), RPB = AW_THREADS / LPR;
  const int lane = threadIdx.x % LPR;
  const int64_t n = p.s.T * p.Hq, i = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
  const int64_t row = min(i, n - 1);  // (whole waves: rows past the last repeat it)
  const int64_t t = row / p.Hq;
  const int h = (int)(row - t * p.Hq), kvh = h / p.G;
  float f[8];
  VecIO<DT>::unpack(reinterpret_cast<const uint4*>(p.q + row * D)[lane], f);
  float safe;
  const uint2 c = row_codes_wide<D>(f, lane, p.rotate, safe);
  if (i >= n) return;
  const int64_t to = ((int64_t)kvh * p.s.T + t) * p.G + h - kvh * p.G;
  reinterpret_cast<uint2*>(p.codes + to * D)[lane] = c;
  if (lane == 0) {
    const float l = p.lse[row];
    // (a row that sees nothing: no weights)
    p.rows[to] = make_float2(safe * p.q_mul, l == -INFINITY ? INFINITY : l * 1.4426950408889634f);
  }
}

template <int D>
__global__ void __launch_bounds__(AW_THREADS) weights_kernel(const WeightArgs p) {
  constexpr int KS = D / 64, KG = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g4 = lane >> 4;
  const int cap = p.s.maxb * p.s.bs;
  for (int64_t id = blockIdx.x;; id += gridDim.x) {
    // the sequence and tile of item id: tiles of all sequences in order, KV heads next to each other
    const int64_t unit = id / p.Hkv;
    const int kvh = (int)(id - unit * p.Hkv);
    int b = -1, tile = 0;
    int64_t before = 0;
    for (int b0 = 0; b0 < p.s.B && b < 0; b0 += 64) {
      const int len = b0 + lane < p.s.B ? min(max(p.s.lens[b0 + lane], 0), cap) : 0;
      int64_t sum = (len + AW_KEYS - 1) / AW_KEYS;
      const int mine = (int)sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int64_t x = __shfl_up(sum, o, 64);
        if (lane >= o) sum += x;
      }
      const uint64_t past = __builtin_amdgcn_ballot_w64(before + sum > unit);
      if (past) {
        const int at = __builtin_ctzll(past);
        b = b0 + at;
        tile = (int)(unit - (before + __shfl(sum, at, 64) - __shfl(mine, at, 64)));
      }
      before += __shfl(sum, 63, 64);
    }
    b = __builtin_amdgcn_readfirstlane(b);
    tile = __builtin_amdgcn_readfirstlane(tile);
    if (b < 0) return;
    const int len = min(max(p.s.lens[b], 0), cap);
    const int64_t row0 = p.s.row(b);
    const int n = max(0, (int)(p.s.row(b + 1) - row0));
    const int64_t pos64 = max((int64_t)p.s.lens[b] - n, (int64_t)-(1 << 28));
    const int pos0 = (int)min(pos64, (int64_t)1 << 30);
    const int key0 = tile * AW_KEYS + wave * 64;
    if (key0 >= len) continue;
    // the wave's keys: group g, key col of it
    v4i ka[KG][KS];
    float ks[KG];
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      const int key = key0 + 16 * g;
      const int j = key / p.s.bs;
      const int blk = key < len ? p.s.block(b, j) : -1;
      ks[g] = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) ka[g][s] = v4i{0, 0, 0, 0};
      if (blk >= 0) {
        const int64_t bh = (int64_t)blk * p.Hkv + kvh;
        ks[g] = p.ks[bh];
        const int8_t* at = p.k + (bh * p.s.bs + key - j * p.s.bs + col) * D + 16 * g4;
#pragma unroll
        for (int s = 0; s < KS; ++s) ka[g][s] = *reinterpret_cast<const v4i*>(at + 64 * s);
      } else {
        ks[g] = -1.f;  // no keys
      }
    }
    // the rows that see any of them: (token, head of the group) in order
    const int64_t t0 = max(0, key0 - pos0);
    const int64_t t1 = p.window < 0 ? n : min((int64_t)n, (int64_t)key0 + 63 + p.window - pos0);
    const int r0 = (int)min(t0, (int64_t)n) * p.G, r1 = (int)max(t1, (int64_t)0) * p.G;
    const int8_t* codes = p.codes + ((int64_t)kvh * p.s.T + row0) * p.G * D;
    const float2* rows = p.rows + ((int64_t)kvh * p.s.T + row0) * p.G;
    float acc[KG][4] = {};
    for (int r = r0; r < r1; r += 16) {
      const int row = min(r + col, r1 - 1);
      v4i qb[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s) qb[s] = *reinterpret_cast<const v4i*>(codes + (int64_t)row * D + 64 * s + 16 * g4);
      const float2 y = rows[row];
      const int pos = pos0 + row / p.G;
      const int lim = r + col < r1 ? pos + 1 : 0;
      const int low = p.window >= 0 ? pos - p.window + 1 : 0;
#pragma unroll
      for (int g = 0; g < KG; ++g) {
        v4i sc = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) sc = __builtin_amdgcn_mfma_i32_16x16x64_i8(ka[g][s], qb[s], sc, 0, 0, 0);
        const float a = y.x * ks[g];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + 16 * g + 4 * g4 + i;
          const float e = __builtin_amdgcn_exp2f(fmaf((float)sc[i], a, -y.y));
          acc[g][i] += key < lim && key >= low && ks[g] >= 0.f ? e : 0.f;
        }
      }
    }
#pragma unroll
    for (int g = 0; g < KG; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) acc[g][i] += __shfl_xor(acc[g][i], o, 64);
    // lane (g4, col) writes key 16 (col / 4) + 4 g4 + col % 4
    float mine = 0.f;
#pragma unroll
    for (int g = 0; g < KG; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (col == 4 * g + i) mine = acc[g][i];
    const int key = key0 + 16 * (col >> 2) + 4 * g4 + (col & 3);
    if (key < len) {
      float* w = p.w + b * p.wb + kvh * p.wh + key;
      *w = (key < pos0 ? *w * p.decay : 0.f) + mine;
    }
  }
}

size_t weights_bytes(int64_t T, int64_t Hq, int64_t D) { return (size_t)(T * Hq) * (D + sizeof(float2)); }

}  // namespace
}  // namespace sl8

using namespace sl8;

extern "C" size_t sl8_attn_weights_block8_workspace(int64_t T, int64_t Hq, int64_t D) {
  if (T <= 0 || Hq <= 0 || D <= 0 || T >= (1LL << 28) || Hq >= (1 << 16) || D > 256) return 0;
  return weights_bytes(T, Hq, D);
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
  SL8_CHECK_ARG(T * Hq < (1LL << 30), "fni8 %s: shape too large", tag);
  if (B == 0 || max_blocks_per_seq == 0) return SL8_OK;
  SL8_CHECK_ARG(context_lens && block_table && weights && (num_blocks == 0 || (k_cache && k_scale)) &&
                    (T == 0 || (q && lse)),
                "fni8 %s: null pointer", tag);
  SL8_CHECK_ARG(aligned(q, 16) && aligned(k_cache, 16), "fni8 %s: q/k_cache must be 16-byte aligned", tag);
  SL8_CHECK_ARG(T == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= weights_bytes(T, Hq, D)),
                "fni8 %s: workspace needs %zu bytes", tag, weights_bytes(T, Hq, D));
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
  p.rows = reinterpret_cast<float2*>(p.codes + T * Hq * D);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t most = B * Hkv * ((max_blocks_per_seq * block_size + AW_KEYS - 1) / AW_KEYS);
  const unsigned grid = (unsigned)std::min<int64_t>(most, (int64_t)cu_count() * 8);
  auto by_d = [&](auto d) {
    constexpr int DD = decltype(d)::value;
    constexpr int RPB = AW_THREADS / row_lanes(DD);
    const unsigned pre = (unsigned)((T * Hq + RPB - 1) / RPB);
    if (T) {
      if (dtype == SL8_DTYPE_F16) weights_rows_kernel<SL8_DTYPE_F16, DD><<<pre, AW_THREADS, 0, st>>>(p);
      else weights_rows_kernel<SL8_DTYPE_BF16, DD><<<pre, AW_THREADS, 0, st>>>(p);
    }
    weights_kernel<DD><<<grid, AW_THREADS, 0, st>>>(p);
  };
  if (D == 64) by_d(std::integral_constant<int, 64>{});
  else if (D == 128) by_d(std::integral_constant<int, 128>{});
  else by_d(std::integral_constant<int, 256>{});
  SL8_CHECK_LAUNCH(tag);
  return SL8_OK;
}
