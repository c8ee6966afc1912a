// Linear layer of int8 weights with a scale per output channel, activations quantised with a scale per
// token (the per_row_i8 weights of the package's containers):
//   xs[m] = amax|x[m]| * fp32(1/127) (1 for a row of zeros), c = clamp(rint(x / xs), -127, 127),
//   y[m,n] = xs[m] * ws[n] * sum_k c[m,k] w[n,k] + bias[n], rounded once.
// The sums are exact integers (K < 2^17).
#include <algorithm>

#include "attn_common.hpp"
#include "rowquant.hpp"

namespace sl8 {
namespace {

constexpr int W8_MAX_K = 1 << 17;

// A row's codes in scratch, [M][Kp]: chunk c holds elements 16 c .. 16 c + 15. Where K is no multiple of
// 16 the last one holds the row's last 16 elements, those of the chunk in front as zeros, so that 16 bytes of
// a weight row that meet it end where the row ends; zeros up to Kp.
struct W8Args {
  const void* x;
  const int8_t* w;
  const float* ws;
  const void* bias;
  void* out;
  int8_t* codes;
  float* xs;
  int M, N, K, Kp;
  int bias_dt;  // -1: none
};

inline int64_t w8_padded(int64_t K) { return (K + 63) / 64 * 64; }

template <int DT>
__global__ void __launch_bounds__(256) w8_quant_kernel(const W8Args p) {
  __shared__ float amax_s[4];
  using T = typename Elem<DT>::T;
  const T* x = static_cast<const T*>(p.x) + (int64_t)blockIdx.x * p.K;
  float amax = 0.f;
  for (int i = threadIdx.x; i < p.K; i += 256) amax = fmaxf(amax, fabsf(Elem<DT>::ld(x, i)));
  amax = lane_group_max<64>(amax);
  if ((threadIdx.x & 63) == 0) amax_s[threadIdx.x >> 6] = amax;
  __syncthreads();
  amax = fmaxf(fmaxf(amax_s[0], amax_s[1]), fmaxf(amax_s[2], amax_s[3]));
  const float s = amax * (1.0f / 127.0f), safe = s == 0.f ? 1.f : s;
  if (threadIdx.x == 0) p.xs[blockIdx.x] = safe;
  const int whole = p.K & ~15;
  for (int i = threadIdx.x; i < p.Kp; i += 256) {
    int e = i;
    if (i >= whole) e = whole < p.K && i < whole + 16 ? p.K - 16 + i - whole : p.K;
    const bool live = e < p.K && (i < whole || e >= whole);
    p.codes[(int64_t)blockIdx.x * p.Kp + i] = live ? code_of(Elem<DT>::ld(x, e), safe) : 0;
  }
}

typedef v4i v4i_u __attribute__((aligned(4)));  // rows of K % 16 != 0 are 4-byte aligned

__device__ __forceinline__ float w8_bias(const W8Args& p, int n) {
  if (p.bias_dt < 0) return 0.f;
  if (p.bias_dt == SL8_DTYPE_F32) return static_cast<const float*>(p.bias)[n];
  const uint16_t b = static_cast<const uint16_t*>(p.bias)[n];
  return p.bias_dt == SL8_DTYPE_F16 ? h2f(b) : bf2f(b);
}

// A wave has 16 output channels (A operands, straight from memory) of 16 tokens.
template <int ODT>
__global__ void __launch_bounds__(256) w8_gemm_kernel(const W8Args p) {
  const int lane = threadIdx.x & 63, col = lane & 15, g4 = lane >> 4;
  const int n0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 16, m0 = blockIdx.y * 16;
  if (n0 >= p.N) return;
  const int8_t* w = p.w + (int64_t)min(n0 + col, p.N - 1) * p.K;
  const int8_t* x = p.codes + (int64_t)min(m0 + col, p.M - 1) * p.Kp + 16 * g4;
  v4i acc = {0, 0, 0, 0};
  for (int k = 0; k < p.K; k += 64) {
    const v4i a = *reinterpret_cast<const v4i_u*>(w + min(k + 16 * g4, p.K - 16));
    const v4i b = *reinterpret_cast<const v4i*>(x + k);
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, acc, 0, 0, 0);
  }
  const int m = m0 + col;
  if (m >= p.M) return;
  const float xs = p.xs[m];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = n0 + 4 * g4 + i;
    if (n < p.N) st_out<ODT>(p.out, (int64_t)m * p.N + n, (float)acc[i] * xs * p.ws[n] + w8_bias(p, n));
  }
}

size_t w8_bytes(int64_t M, int64_t K) { return (size_t)M * (w8_padded(K) + sizeof(float)); }

}  // namespace
}  // namespace sl8

using namespace sl8;

extern "C" size_t sl8_linear_w8a8_workspace(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || M >= (1LL << 31) || N >= (1LL << 31) || K >= W8_MAX_K) return 0;
  return w8_bytes(M, K);
}

extern "C" int sl8_linear_w8a8(const void* x, int x_dtype, const int8_t* w, const float* w_scale, const void* bias,
                               int bias_dtype, void* out, int out_dtype, int64_t M, int64_t N, int64_t K,
                               void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  const char* tag = "linear_w8a8";
  auto known = [](int dt) { return dt == SL8_DTYPE_F16 || dt == SL8_DTYPE_BF16 || dt == SL8_DTYPE_F32; };
  SL8_CHECK_ARG(known(x_dtype), "fni8 %s: x must be float16/bfloat16/float32", tag);
  SL8_CHECK_ARG(known(out_dtype), "fni8 %s: out_dtype must be float16/bfloat16/float32", tag);
  SL8_CHECK_ARG(!bias || known(bias_dtype), "fni8 %s: bias must be float16/bfloat16/float32", tag);
  SL8_CHECK_ARG(M >= 0 && N >= 0 && M < (1LL << 31) && N < (1LL << 31), "fni8 %s: bad shape", tag);
  SL8_CHECK_ARG(K >= 16 && K % 4 == 0 && K < W8_MAX_K,
                "fni8 %s: K must be a multiple of 4, 16 to %d, got %lld", tag, W8_MAX_K - 4, (long long)K);
  if (M == 0 || N == 0) return SL8_OK;
  SL8_CHECK_ARG(x && w && w_scale && out, "fni8 %s: null pointer", tag);
  SL8_CHECK_ARG(aligned(w, K % 16 ? 4 : 16), "fni8 %s: w must be 16-byte aligned (4 where K %% 16 != 0)", tag);
  SL8_CHECK_ARG(workspace && aligned(workspace, 16) && workspace_bytes >= w8_bytes(M, K),
                "fni8 %s: workspace needs %zu bytes", tag, w8_bytes(M, K));
  W8Args p{};
  p.x = x; p.w = w; p.ws = w_scale; p.bias = bias; p.out = out;
  p.bias_dt = bias ? bias_dtype : -1;
  p.M = (int)M; p.N = (int)N; p.K = (int)K; p.Kp = (int)w8_padded(K);
  p.codes = static_cast<int8_t*>(workspace);
  p.xs = reinterpret_cast<float*>(p.codes + M * p.Kp);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  SL8_CHECK_ARG(M < (1LL << 24) && (M + 15) / 16 < 65536, "fni8 %s: shape too large", tag);
  if (x_dtype == SL8_DTYPE_F16) w8_quant_kernel<SL8_DTYPE_F16><<<(unsigned)M, 256, 0, st>>>(p);
  else if (x_dtype == SL8_DTYPE_BF16) w8_quant_kernel<SL8_DTYPE_BF16><<<(unsigned)M, 256, 0, st>>>(p);
  else w8_quant_kernel<SL8_DTYPE_F32><<<(unsigned)M, 256, 0, st>>>(p);
  const dim3 grid((unsigned)((N + 63) / 64), (unsigned)((M + 15) / 16));
  if (out_dtype == SL8_DTYPE_F16) w8_gemm_kernel<SL8_DTYPE_F16><<<grid, 256, 0, st>>>(p);
  else if (out_dtype == SL8_DTYPE_BF16) w8_gemm_kernel<SL8_DTYPE_BF16><<<grid, 256, 0, st>>>(p);
  else w8_gemm_kernel<SL8_DTYPE_F32><<<grid, 256, 0, st>>>(p);
  SL8_CHECK_LAUNCH(tag);
  return SL8_OK;
}
