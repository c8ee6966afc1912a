// Rotary positions of Q and K in one launch (rope.hpp: the mathematics and the row code). No
// counterpart in the reference, whose callers rotate before they quantise.
//
// Bound by the bytes: every row is read and written once, 16 bytes an access, and a thread keeps its
// pairs' angles over the heads, so that the table and the positions are read once a token. 6121
// tokens of 32 + 8 heads, D = 128, bf16, three axes (129 MB): 25.2 us, 5.1 TB/s, the rate of a
// copy; 4 x 4096 tokens of 16 + 16 heads, D = 80, fp32 (341 MB): 73.6 us, 4.6 TB/s (88 with 8-byte
// accesses). 64 tokens (1.3 MB): 5.8 us, the chain position, angles, rows (loaded behind the angles), store. Two heads of a thread in
// flight at once are slower (26.7 us for the 25.2 above: more registers, fewer waves).
#include "rope.hpp"

namespace sl8 {
namespace {

constexpr int ROPE_THREADS = 256;

template <int DT, int N>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(const RopeArgs a, const RopeRows t) {
  rope_block<DT, N>(a, t, blockIdx.x);
}

}  // namespace
}  // namespace sl8

using namespace sl8;

extern "C" int sl8_rope(const void* q, const void* k, int dtype, int64_t q_stride_b, int64_t q_stride_h,
                        int64_t q_stride_s, int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_s,
                        const void* positions, int positions_i64, int64_t pos_axis, int64_t pos_b,
                        const float* table, int64_t table_rows, const int32_t* sections, int axes,
                        int interleaved, int inverse, void* q_out, void* k_out, int64_t B, int64_t Hq,
                        int64_t Hkv, int64_t S, int64_t D, int64_t R, void* stream) {
  clear_error();
  SL8_CHECK_ARG(dtype == SL8_DTYPE_F16 || dtype == SL8_DTYPE_BF16 || dtype == SL8_DTYPE_F32,
                "fni8 rope: q/k must be float16/bfloat16/float32");
  SL8_CHECK_ARG(B >= 0 && Hq >= 0 && Hkv >= 0 && S >= 0, "fni8 rope: bad shape");
  SL8_CHECK_ARG(D >= 2 && D % 2 == 0 && D <= 512, "fni8 rope: head dim must be even, 2..512, got %lld",
                (long long)D);
  SL8_CHECK_ARG(Hq + Hkv < (1 << 20) && S < (1LL << 31) && B < (1LL << 31) && B * S < (1LL << 31),
                "fni8 rope: shape too large");
  if (B * S * (Hq + Hkv) == 0) return SL8_OK;
  RopeArgs a;
  if (const int rc = rope_args("rope", a, positions, positions_i64, pos_axis, pos_b, table, table_rows,
                               R, D, sections, axes, interleaved, inverse)) return rc;
  SL8_CHECK_ARG((Hq == 0 || (q && q_out)) && (Hkv == 0 || (k && k_out)),
                "fni8 rope: null pointer");
  RopeRows t{q, k, q_out, k_out, {q_stride_b, q_stride_h, q_stride_s}, {k_stride_b, k_stride_h, k_stride_s},
             {Hq * S * D, S * D, D}, {Hkv * S * D, S * D, D}, B * S, S, (int)Hq, (int)Hkv, (int)D, 1, 1};
  const void* ptrs[4];
  int64_t strides[6];
  int np = 0, ns = 0;
  if (Hq) ptrs[np++] = q, ptrs[np++] = q_out;
  if (Hkv) ptrs[np++] = k, ptrs[np++] = k_out;
  for (int i = 0; i < 3; ++i) {
    if (Hq) strides[ns++] = t.qs[i];
    if (Hkv) strides[ns++] = t.ks[i];
  }
  const int n = rope_pairs(D, R, dtype, ptrs, np, strides, ns);
  rope_shape(t, ROPE_THREADS / (int)(D / (2 * n)));
  const int64_t grid = (t.T + t.tokens - 1) / t.tokens;
  SL8_CHECK_ARG(grid < (1LL << 32) / ROPE_THREADS, "fni8 rope: shape too large");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  auto by_n = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (n == 8) rope_kernel<DT, 8><<<(unsigned)grid, ROPE_THREADS, 0, st>>>(a, t);
    else if (n == 4) rope_kernel<DT, 4><<<(unsigned)grid, ROPE_THREADS, 0, st>>>(a, t);
    else rope_kernel<DT, 1><<<(unsigned)grid, ROPE_THREADS, 0, st>>>(a, t);
  };
  if (dtype == SL8_DTYPE_F16) by_n(std::integral_constant<int, SL8_DTYPE_F16>{});
  else if (dtype == SL8_DTYPE_BF16) by_n(std::integral_constant<int, SL8_DTYPE_BF16>{});
  else by_n(std::integral_constant<int, SL8_DTYPE_F32>{});
  SL8_CHECK_LAUNCH("rope");
  return SL8_OK;
}
