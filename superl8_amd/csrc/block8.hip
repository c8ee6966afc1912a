// Append of new tokens to the block-scaled paged int8 cache (block8.hpp), K turned by position on
// the way, with the turned Q of the same tokens. No counterpart in the reference, whose paged
// cache has a scale per token.
//
// A block and head that gets new rows takes the scale
//   s' = max(s of the rows that it keeps, amax|new rows| * fp32(1/127), 2^-60)
// and holds rint(x / s') of the new rows; kept codes c become rint(c * (s / s')) where s grew. Rows
// behind the last new one stay as they are: they are not read before they are written. The least
// scale keeps the reciprocals that the attention sums within 32 bits.
//
// One workgroup per (block, head, K or V): it owns the block's scale, so nothing is shared or
// atomic. It holds its rows in registers between the maximum and the codes, 8 elements a thread,
// D / 8 threads a row. 7312 tokens of four prompts, 32 / 8 heads, D = 128, bf16, three position
// axes, Q with them (165 MB): 43 to 45 us, 3.7 TB/s. The bytes alone would take 32; what bounds it is the
// chain of each workgroup (offsets and lengths, rows beside the block id, then for each pass over them the
// positions and after those the angles, maximum, barrier, codes) at four waves a SIMD (104 registers),
// with VALU busy in 64 % of the cycles, most of it the Hadamard rotation (25 instructions an element of K, 7 of V).
// Held to 96 or 80 registers it spills (101, 113 us with the 42 of reading the values back, against
// 93); workgroups of 512 or 1024 threads wait longer at the barrier (kernel 53, 61 against 47 then). A decode
// step of 32 sequences (0.7 MB): 5.7 us, that chain once.
#include "block8.hpp"
#include "rope.hpp"

namespace sl8 {
namespace {

constexpr int APP_THREADS = 256;

struct AppendArgs {
  Block8Seqs s;
  const void *k, *v;
  int64_t kst[2], vst[2];  // strides of token and head
  int8_t *k_cache, *v_cache;
  float *k_scale, *v_scale;
  int Hkv;
  bool rope;
  bool has_q;
  uint32_t share;  // with Q: the part of the workgroups that have blocks (32 fraction bits)
};

// Elements 8 lane .. 8 lane + 7 of a row held by LPR lanes, turned.
template <int LPR>
__device__ __forceinline__ void rope_row(const RopeArgs& a, int64_t token, float* f, int lane) {
  const int i0 = 8 * lane, half = a.R / 2;
  if (a.interleaved) {
    if (i0 < a.R) {
      float c[4], s[4];
      rope_angles<4>(a, token, i0 / 2, c, s);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float u = f[2 * e], v = f[2 * e + 1];
        f[2 * e] = u * c[e] - v * s[e];
        f[2 * e + 1] = v * c[e] + u * s[e];
      }
    }
    return;
  }
  const bool low = i0 < half;
  const int mate = low ? lane + half / 8 : i0 < a.R ? lane - half / 8 : lane;
  float o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = __shfl(f[e], mate, LPR);
  if (i0 < a.R) {
    float c[8], s[8];
    rope_angles<8>(a, token, low ? i0 : i0 - half, c, s);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = low ? f[e] * c[e] - o[e] * s[e] : f[e] * c[e] + o[e] * s[e];
  }
}

// NP: passes of 256 threads over the rows of a block.
template <int DT, int D, int NP, bool ROT>
__global__ void __launch_bounds__(APP_THREADS)
append_block8_kernel(const AppendArgs p, const RopeArgs a, const RopeRows q) {
  // workgroups of blocks and of Q by turns: the former wait for chains of loads while the latter stream
  const uint32_t wg = __umulhi(blockIdx.x, p.share), next = __umulhi(blockIdx.x + 1, p.share);
  if (p.has_q && wg == next) return rope_block<DT, 8>(a, q, blockIdx.x - wg);
  const uint32_t page = p.has_q ? wg : blockIdx.x;
  constexpr int LPR = D / 8, RPB = APP_THREADS / LPR;
  __shared__ float amax_s[APP_THREADS / 64];
  const Block8Seqs& s = p.s;
  const int lane = threadIdx.x % LPR, r0 = threadIdx.x / LPR;
  const bool is_v = page & 1;
  const int h = (page >> 1) % p.Hkv, unit = (page >> 1) / p.Hkv;

  // (rows / bs + 2: at least as many units as blocks that n rows can touch)
  const Seq q0 = s.cu ? seq_of(s, threadIdx.x & 63, unit, [&](int row0, int b) { return row0 / s.bs + 2 * b; })
                      : Seq{unit, unit, unit < s.B ? 1 : 0, unit < s.B ? s.lens[unit] : 0, 0};
  if (q0.n <= 0 || q0.len < q0.n) return;
  const int start = q0.len - q0.n;
  const int pg = start / s.bs + q0.nth;
  if (pg >= s.maxb) return;
  const int lo = max(start, pg * s.bs), hi = min(q0.len, (pg + 1) * s.bs);
  if (lo >= hi) return;
  const int id = s.block(q0.b, pg);
  const int off = lo - pg * s.bs, cnt = hi - lo;
  const int64_t tok = q0.row0 + (lo - start);
  const void* x = is_v ? p.v : p.k;
  const int64_t st = is_v ? p.vst[0] : p.kst[0], sh = is_v ? p.vst[1] : p.kst[1];

  // all rows' loads go out before the first is used and beside the block's; rows past the last repeat it
  uint4 raw[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i)
    if (NP <= 4 || i * RPB < cnt)
      raw[i] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) +
                                               (tok + min(i * RPB + r0, cnt - 1)) * st + h * sh + 8 * lane);
  if (id < 0) return;
  const int64_t bh = (int64_t)id * p.Hkv + h;
  int8_t* cache = (is_v ? p.v_cache : p.k_cache) + bh * s.bs * D;
  float* scale = (is_v ? p.v_scale : p.k_scale) + bh;
  const float old = off ? *scale : 0.f;

  float f[NP][8];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    if (i * RPB >= cnt) break;
    VecIO<DT>::unpack(raw[i], f[i]);
    if (!is_v) {
      if (p.rope) rope_row<LPR>(a, tok + min(i * RPB + r0, cnt - 1), f[i], lane);
      if constexpr (ROT) hadamard_row<D, DT != SL8_DTYPE_F16>(f[i], lane);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(f[i][e]));
  }
  amax = lane_group_max<64>(amax);
  if ((threadIdx.x & 63) == 0) amax_s[threadIdx.x / 64] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < APP_THREADS / 64; ++w) amax = fmaxf(amax, amax_s[w]);
  const float now = fmaxf(fmaxf(old, amax * (1.0f / 127.0f)), 0x1p-60f);

#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = i * RPB + r0;
    if (r < cnt) *reinterpret_cast<uint2*>(cache + (int64_t)(off + r) * D + 8 * lane) = codes8(f[i], now);
  }
  if (off && now != old) {
    const float ratio = __fdiv_rn(old, now);
    for (int r = r0; r < off; r += RPB) {
      uint2* c = reinterpret_cast<uint2*>(cache + (int64_t)r * D + 8 * lane);
      const uint2 w = *c;
      uint32_t o[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int8_t v = (int8_t)((e < 4 ? w.x : w.y) >> (8 * (e % 4)));
        o[e / 4] |= (uint32_t)(uint8_t)(int8_t)rintf((float)v * ratio) << (8 * (e % 4));
      }
      *c = make_uint2(o[0], o[1]);
    }
  }
  if (threadIdx.x == 0) *scale = now;
}

}  // namespace
}  // namespace sl8

using namespace sl8;

extern "C" int sl8_kv_append_block8(const void* k_new, const void* v_new, const void* q, int dtype,
                                    int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t,
                                    int64_t v_stride_h, int64_t q_stride_t, int64_t q_stride_h,
                                    const void* positions, int positions_i64, const float* table, int64_t table_rows,
                                    const int32_t* sections, int axes, int interleaved, int rotate,
                                    const int32_t* cu_lens, const int32_t* context_lens,
                                    const int32_t* block_table, int8_t* k_cache, float* k_scale,
                                    int8_t* v_cache, float* v_scale, void* q_out, int64_t T,
                                    int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t R,
                                    int64_t num_blocks, int64_t block_size, int64_t max_blocks_per_seq,
                                    void* stream) {
  clear_error();
  const char* tag = "kv_append_block8";
  SL8_CHECK_ARG(dtype == SL8_DTYPE_F16 || dtype == SL8_DTYPE_BF16,
                "fni8 %s: q/k_new/v_new must be float16 or bfloat16", tag);
  SL8_CHECK_ARG(T >= 0 && T < (1LL << 28) && B >= 0 && B < (1 << 24) && Hq >= 0 && Hq < (1 << 16) &&
                    num_blocks >= 0 && num_blocks < (1LL << 31) && max_blocks_per_seq >= 0 &&
                    max_blocks_per_seq < (1LL << 31) && block_size >= 0 && block_size < (1 << 16),
                "fni8 %s: shape too large", tag);
  AppendArgs p{};
  p.s = Block8Seqs{cu_lens, context_lens, block_table, T, (int)B, (int)max_blocks_per_seq, (int)num_blocks,
                   (int)block_size};
  if (const int rc = block8_check(tag, p.s, Hkv, D)) return rc;
  RopeArgs a{};
  RopeRows qr{};
  p.rope = positions != nullptr;
  SL8_CHECK_ARG(p.rope || Hq == 0, "fni8 %s: q needs positions", tag);
  if (T == 0) return SL8_OK;
  if (p.rope) {
    if (const int rc = rope_args(tag, a, positions, positions_i64, T, 0, table, table_rows, R, D,
                                 sections, axes, interleaved, 0)) return rc;
    SL8_CHECK_ARG(R % 16 == 0, "fni8 %s: rotary dim must be a multiple of 16, got %lld", tag, (long long)R);
  }
  SL8_CHECK_ARG(k_new && v_new && context_lens &&
                    (max_blocks_per_seq == 0 || block_table) &&
                    (num_blocks == 0 || (k_cache && k_scale && v_cache && v_scale)) &&
                    (Hq == 0 || (q && q_out)),
                "fni8 %s: null pointer", tag);
  const bool ok = aligned(k_new, 16) && aligned(v_new, 16) && aligned(q, 16) && aligned(q_out, 16) &&
                  aligned(k_cache, 8) && aligned(v_cache, 8) &&
                  (k_stride_t | k_stride_h | v_stride_t | v_stride_h | (Hq ? q_stride_t | q_stride_h : 0)) % 8 == 0;
  SL8_CHECK_ARG(ok, "fni8 %s: rows must be 16-byte aligned", tag);
  p.kst[0] = k_stride_t; p.kst[1] = k_stride_h;
  p.vst[0] = v_stride_t; p.vst[1] = v_stride_h;
  p.k = k_new; p.v = v_new;
  p.k_cache = k_cache; p.v_cache = v_cache; p.k_scale = k_scale; p.v_scale = v_scale;
  p.Hkv = (int)Hkv;
  const int64_t units = cu_lens ? T / block_size + 2 * B : B;
  const int64_t page_wgs = num_blocks ? units * Hkv * 2 : 0;
  int64_t q_wgs = 0;
  if (Hq) {
    qr = RopeRows{q, nullptr, q_out, nullptr, {0, q_stride_h, q_stride_t}, {}, {0, D, Hq * D}, {}, T, T,
                  (int)Hq, 0, (int)D, 1, 1};
    rope_shape(qr, APP_THREADS / (int)(D / 16));
    q_wgs = (T + qr.tokens - 1) / qr.tokens;
  }
  const int64_t grid = page_wgs + q_wgs;
  if (grid == 0) return SL8_OK;
  SL8_CHECK_ARG(grid < (1LL << 32) / APP_THREADS, "fni8 %s: shape too large", tag);
  // ceil(2^32 page_wgs / grid): workgroup i has (i share) >> 32 of blocks before it, all of them page_wgs
  p.has_q = q_wgs > 0;
  p.share = p.has_q ? (uint32_t)((((uint64_t)page_wgs << 32) + grid - 1) / grid) : 0;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  using std::integral_constant;
  auto go = [&](auto dt, auto d, auto np) {
    constexpr int DT = decltype(dt)::value, DD = decltype(d)::value, NP = decltype(np)::value;
    if (rotate) append_block8_kernel<DT, DD, NP, true><<<(unsigned)grid, APP_THREADS, 0, st>>>(p, a, qr);
    else append_block8_kernel<DT, DD, NP, false><<<(unsigned)grid, APP_THREADS, 0, st>>>(p, a, qr);
  };
  auto by_np = [&](auto dt, auto d) {  // passes that the rows of a block take, to a power of two
    const int64_t np = (block_size * decltype(d)::value / 8 + APP_THREADS - 1) / APP_THREADS;
    if (np <= 1) go(dt, d, integral_constant<int, 1>{});
    else if (np <= 4) go(dt, d, integral_constant<int, 4>{});
    else if constexpr (decltype(d)::value > 64) go(dt, d, integral_constant<int, decltype(d)::value / 16>{});
  };
  auto by_d = [&](auto dt) {
    if (D == 64) by_np(dt, integral_constant<int, 64>{});
    else if (D == 128) by_np(dt, integral_constant<int, 128>{});
    else by_np(dt, integral_constant<int, 256>{});
  };
  if (dtype == SL8_DTYPE_F16) by_d(integral_constant<int, SL8_DTYPE_F16>{});
  else by_d(integral_constant<int, SL8_DTYPE_BF16>{});
  SL8_CHECK_LAUNCH(tag);
  return SL8_OK;
}
