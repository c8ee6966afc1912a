// Attention of new tokens over the block-scaled paged int8 cache (block8.hpp). No counterpart in
// the reference, whose paged cache has a scale per token and one query token per sequence.
//
// Query row i of a sequence's n new ones stands at position p = len - n + i and sees keys j <= p,
// with a window j > p - window too. Its row (rotated by the Hadamard matrix as the keys were, in
// 32 bits) is quantised to int8 with one scale qs; then
//   s_j = qs * scale * log2(e) * ks[block(j)] * <q, k_j> (exact integers inside),
//   out = sum_j 2^(s_j - m) vs[block(j)] v_j / sum_j 2^(s_j - m);
// a row that sees nothing gives zeros.
#include "block8.hpp"
#include "rowquant.hpp"

namespace sl8 {
namespace {

struct AttnArgs {
  Block8Seqs s;
  const uint16_t* q;
  const int8_t *k, *v;
  const float *ks, *vs;
  void* out;
  int Hq, Hkv;
  float q_mul;
  int64_t window;
};

// One wave per query row and head: a lane is a key in the scores, D / 64 channels in the sum.
template <int DT, int D, bool ROT>
__global__ void __launch_bounds__(64) attn_block8_row_kernel(const AttnArgs p) {
  constexpr int LPR = row_lanes(D), C = D / 64;
  __shared__ __attribute__((aligned(16))) int q_s[D / 4];
  __shared__ float w_s[64];
  const Block8Seqs& s = p.s;
  const int lane = threadIdx.x;
  const int64_t t = blockIdx.x / p.Hq;
  const int h = blockIdx.x % p.Hq, kvh = h / (p.Hq / p.Hkv);
  const int64_t to = (t * p.Hq + h) * D;

  const int b = seq_of(s.B, lane, t, [&](int i) { return s.row(i); });
  int64_t lo = 0, hi = 0;
  if (b >= 0 && t < s.row(b + 1)) {
    const int64_t len = s.lens[b], pos = len - (s.row(b + 1) - s.row(b)) + (t - s.row(b));
    hi = min(min(pos + 1, len), (int64_t)s.maxb * s.bs);
    if (p.window >= 0) lo = max((int64_t)0, pos - p.window + 1);
  }

  float f[8] = {};
  if (lane < LPR) VecIO<DT>::unpack(reinterpret_cast<const uint4*>(p.q + to)[lane], f);
  if constexpr (ROT) hadamard_row<D, DT != SL8_DTYPE_F16>(f, lane);
  float amax = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(f[e]));
  amax = lane_group_max<LPR>(amax);
  const float sc = amax * (1.0f / 127.0f), safe = sc == 0.f ? 1.f : sc;
  if (lane < LPR) reinterpret_cast<uint2*>(q_s)[lane] = row_codes8<DT>(f, safe);
  const float qs = __shfl(safe, 0, 64) * p.q_mul;
  __syncthreads();

  float m = -1e30f, l = 0.f, o[C] = {};
  for (int64_t j0 = lo; j0 < hi; j0 += 64) {
    const int64_t j = j0 + lane;
    const int id = j < hi ? s.block(b, (int)(j / s.bs)) : -1;
    float x = -INFINITY, v = 0.f;
    if (id >= 0) {
      const int64_t bh = (int64_t)id * p.Hkv + kvh;
      const int* kr = reinterpret_cast<const int*>(p.k + (bh * s.bs + j % s.bs) * D);
      int acc = 0;
#pragma unroll
      for (int c = 0; c < D / 4; ++c) acc = __builtin_amdgcn_sdot4(kr[c], q_s[c], acc, false);
      x = (float)acc * (qs * p.ks[bh]);
      v = p.vs[bh];
    }
    const float mn = fmaxf(m, wave_max(x));
    const float w = exp2f(x - mn), r = exp2f(m - mn);
    m = mn;
    l = l * r + wave_sum(w);
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] *= r;
    w_s[lane] = id >= 0 ? w * v : 0.f;
    __syncthreads();
    for (int i = 0; i < 64 && j0 + i < hi; ++i) {
      const int ib = s.block(b, (int)((j0 + i) / s.bs));
      if (ib < 0) continue;
      const int8_t* vr = p.v + (((int64_t)ib * p.Hkv + kvh) * s.bs + (j0 + i) % s.bs) * D;
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] = fmaf(w_s[i], (float)vr[lane + 64 * c], o[c]);
    }
    __syncthreads();
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) st_out<DT>(p.out, to + lane + 64 * c, o[c] * inv);
}

}  // namespace
}  // namespace sl8

using namespace sl8;

extern "C" int sl8_attn_paged_block8(const void* q, int dtype, int rotate, float q_scale_mul,
                                     const int8_t* k_cache, const float* k_scale,
                                     const int8_t* v_cache, const float* v_scale,
                                     const int32_t* cu_lens, const int32_t* context_lens,
                                     const int32_t* block_table, void* out, int64_t T, int64_t B,
                                     int64_t Hq, int64_t Hkv, int64_t D, int64_t num_blocks,
                                     int64_t block_size, int64_t max_blocks_per_seq,
                                     int64_t window_left, void* stream) {
  clear_error();
  const char* tag = "attn_paged_block8";
  SL8_CHECK_ARG(dtype == SL8_DTYPE_F16 || dtype == SL8_DTYPE_BF16, "fni8 %s: q must be float16 or bfloat16", tag);
  SL8_CHECK_ARG(T >= 0 && T < (1LL << 28) && B >= 0 && B < (1 << 24) && Hq >= 0 && Hq < (1 << 16) &&
                    num_blocks >= 0 && num_blocks < (1LL << 31) && max_blocks_per_seq >= 0 &&
                    max_blocks_per_seq < (1LL << 31) && block_size >= 0 && block_size < (1 << 16),
                "fni8 %s: shape too large", tag);
  AttnArgs p{Block8Seqs{cu_lens, context_lens, block_table, T, (int)B, (int)max_blocks_per_seq,
                        (int)num_blocks, (int)block_size},
             static_cast<const uint16_t*>(q), k_cache, v_cache, k_scale, v_scale, out, (int)Hq, (int)Hkv,
             q_scale_mul, window_left};
  if (const int rc = block8_check(tag, p.s, Hkv, D)) return rc;
  SL8_CHECK_ARG(Hq % Hkv == 0, "fni8 %s: H_q must be divisible by H_kv (GQA)", tag);
  if (T == 0 || Hq == 0) return SL8_OK;
  SL8_CHECK_ARG(q && out && (B == 0 || (context_lens && (max_blocks_per_seq == 0 || block_table))) &&
                    (num_blocks == 0 || (k_cache && k_scale && v_cache && v_scale)),
                "fni8 %s: null pointer", tag);
  SL8_CHECK_ARG(aligned(q, 16) && aligned(out, 16) && aligned(k_cache, 16) && aligned(v_cache, 16),
                "fni8 %s: q/k_cache/v_cache must be 16-byte aligned", tag);
  SL8_CHECK_ARG(T * Hq < (1LL << 31), "fni8 %s: shape too large", tag);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  using std::integral_constant;
  auto go = [&](auto dt, auto d) {
    constexpr int DT = decltype(dt)::value, DD = decltype(d)::value;
    if (rotate) attn_block8_row_kernel<DT, DD, true><<<(unsigned)(T * Hq), 64, 0, st>>>(p);
    else attn_block8_row_kernel<DT, DD, false><<<(unsigned)(T * Hq), 64, 0, st>>>(p);
  };
  auto by_d = [&](auto dt) {
    if (D == 64) go(dt, integral_constant<int, 64>{});
    else if (D == 128) go(dt, integral_constant<int, 128>{});
    else go(dt, integral_constant<int, 256>{});
  };
  if (dtype == SL8_DTYPE_F16) by_d(integral_constant<int, SL8_DTYPE_F16>{});
  else by_d(integral_constant<int, SL8_DTYPE_BF16>{});
  SL8_CHECK_LAUNCH(tag);
  return SL8_OK;
}
