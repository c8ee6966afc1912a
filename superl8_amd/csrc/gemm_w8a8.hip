// Linear layer of int8 weights with a scale per output channel, activations quantised with a scale per
// token (the per_row_i8 weights of the package's containers):
//   xs[m] = amax|x[m]| * fp32(1/127) (1 for a row of zeros), c = clamp(rint(x / xs), -127, 127),
//   y[m,n] = xs[m] * ws[n] * sum_k c[m,k] w[n,k] + bias[n].
// The sums are exact integers (K < 2^17); scales and bias are applied in fp32, and that is rounded to y's type.
//
// Up to some tens of rows are bound by the weights' bytes, more by the matrix instructions. A call among others (us; a
// copy's 5.16 TB/s and a large int8 product's 2.10 POP/s give the floor): 1 row, 4096 x 4096 9.0 (floor 3.3; one
// kernel); 16 rows, 17408 x 5120 24.4 (17.4); 333 rows, 5003 x 2052 19.4 (3.6: a chain of 17 stages); 4096 rows,
// 17408 x 5120 368 (348). Their kernels in a trace of 30 calls, where clocks differ from those of a long run and a
// kernel's time holds its own launch, so that they do not add up to a call: stream 8.8 to 9.1; codes 4.1, tiles of 32 rows
// 16.2 (5.5 TB/s); codes 4.2, tiles of 64 rows 16.6; codes 19 to 22, tiles of 256 rows 331 to 362, join 16.
#include <algorithm>
#include <cmath>

#include "attn_common.hpp"
#include "rowquant.hpp"

namespace sl8 {
namespace {

constexpr int W8_MAX_K = 1 << 17;
constexpr int W8_BK = 128;     // what a row's codes are padded to
constexpr int W8_STREAM_ROWS = 16, W8_STREAM_K = 5120;  // the most that the streaming kernel takes

// The rows' codes in scratch, [Kp / 128][M16][128]: the rows that meet at a step of K are next to each other,
// in whole lines (rows K bytes apart can have all their lines in a few channels of the L2). Chunk c of a row
// holds elements 16 c .. 16 c + 15. Where K is no multiple of 16 the last one holds the row's last 16 elements,
// those of the chunk in front as zeros, so that 16 bytes of a weight row that meet it end where the row ends;
// zeros up to Kp. Rows from M to M16 are not written: what they meet is not kept.
struct W8Args {
  const void* x;
  const int8_t* w;
  const float* ws;
  const void* bias;
  void* out;
  int8_t* codes;
  float* xs;
  v4i* part;  // sums of the tiles that are split over K
  int M, N, K, Kp;
  int M16;  // M in whole 16s
  int bias_dt;  // -1: none
  int nt_m, nt_n, whole, splits;  // tiles; those before `whole` are not split
};

inline int64_t w8_padded(int64_t K) { return (K + W8_BK - 1) / W8_BK * W8_BK; }

// Four elements of a row (K % 4 == 0: they are aligned).
template <int DT>
__device__ __forceinline__ void w8_ld4(const void* x, int64_t i, float* f) {
  if constexpr (DT == SL8_DTYPE_F32) {
    VecIO<DT>::unpack(*reinterpret_cast<const uint4*>(static_cast<const float*>(x) + i), f);
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(x) + i);
    f[0] = u16_to_f<DT>(v.x & 0xFFFF); f[1] = u16_to_f<DT>(v.x >> 16);
    f[2] = u16_to_f<DT>(v.y & 0xFFFF); f[3] = u16_to_f<DT>(v.y >> 16);
  }
}

// The larger magnitude, by its bits: infinity above all numbers and NaN above that, so that rows which hold one
// come out as such (their scale is not finite) and not as the rest of the row.
__device__ __forceinline__ float w8_top(float amax, float x) {
  return __uint_as_float(max(__float_as_uint(amax), __float_as_uint(x) & 0x7FFFFFFFu));
}

// Chunk c of a row, as above.
template <int DT>
__device__ __forceinline__ void w8_chunk(const W8Args& p, int64_t row, int c, float* f) {
  const bool part = 16 * c + 16 > p.K;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int e = (part ? p.K - 16 : 16 * c) + 4 * j;
    if (16 * c < p.K && e >= 16 * c) w8_ld4<DT>(p.x, row * p.K + e, f + 4 * j);
    else f[4 * j] = f[4 * j + 1] = f[4 * j + 2] = f[4 * j + 3] = 0.f;
  }
}

// The same of a 16-bit row as it is; chunks past the row's last are zeros.
__device__ __forceinline__ void w8_raw(const W8Args& p, int row, int c, uint2* r) {
  const bool part = 16 * c + 16 > p.K;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int e = (part ? p.K - 16 : 16 * c) + 4 * j;
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.x) + (int64_t)row * p.K + e);
    r[j] = 16 * c < p.K && e >= 16 * c ? v : make_uint2(0, 0);
  }
}

// A workgroup a row, 16 elements a thread and pass; NV passes stay in registers between the maximum and the
// codes (0: rows too long for that are read twice).
template <int DT, int NV>
__global__ void __launch_bounds__(256) w8_quant_kernel(const W8Args p) {
  __shared__ float amax_s[4];
  const int64_t row = blockIdx.x;
  const int chunks = p.Kp / 16;
  float f[NV ? NV : 1][16], amax = 0.f;
  auto top = [&](const float* x) {
#pragma unroll
    for (int e = 0; e < 16; ++e) amax = w8_top(amax, x[e]);
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) w8_chunk<DT>(p, row, threadIdx.x + 256 * i, f[i]);
#pragma unroll
    for (int i = 0; i < NV; ++i) top(f[i]);
  } else {
    for (int c = threadIdx.x; c < chunks; c += 256) {
      w8_chunk<DT>(p, row, c, f[0]);
      top(f[0]);
    }
  }
  amax = lane_group_max<64>(amax);
  if ((threadIdx.x & 63) == 0) amax_s[threadIdx.x >> 6] = amax;
  __syncthreads();
  amax = w8_top(w8_top(amax_s[0], amax_s[1]), w8_top(amax_s[2], amax_s[3]));
  const float s = amax * (1.0f / 127.0f), safe = s == 0.f ? 1.f : s;
  if (threadIdx.x == 0) p.xs[row] = safe;
  auto put = [&](int c, const float* x) {
    const uint2 lo = row_codes8<DT>(x, safe), hi = row_codes8<DT>(x + 8, safe);
    if (c < chunks) *reinterpret_cast<uint4*>(p.codes + ((int64_t)(c >> 3) * p.M16 + row) * 128 + 16 * (c & 7)) = make_uint4(lo.x, lo.y, hi.x, hi.y);
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) put(threadIdx.x + 256 * i, f[i]);
  } else {
    for (int c0 = 0; c0 < chunks; c0 += 256) {
      w8_chunk<DT>(p, row, c0 + threadIdx.x, f[0]);
      put(c0 + threadIdx.x, f[0]);
    }
  }
}

// A barrier behind which the workgroup's copies have arrived but for the last N of each thread, and the reads
// in front of it are done. (A fence would wait for all copies.)
template <int N> __device__ __forceinline__ void w8_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);  // vmcnt(N) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

typedef v4i v4i_u __attribute__((aligned(4)));  // rows of K % 16 != 0 are 4-byte aligned

__device__ __forceinline__ float w8_bias(const W8Args& p, int n) {
  if (p.bias_dt < 0) return 0.f;
  if (p.bias_dt == SL8_DTYPE_F32) return static_cast<const float*>(p.bias)[n];
  const uint16_t b = static_cast<const uint16_t*>(p.bias)[n];
  return p.bias_dt == SL8_DTYPE_F16 ? h2f(b) : bf2f(b);
}

// An output in fp32. (A value of its own: where the compiler joins the fma with the conversion to fp16, as it did for
// some elements of the tiles, that rounds once and not twice, and a row's bits went by how the call was cut.)
__device__ __forceinline__ float w8_value(int y, float xs, float ws, float bias) {
  float z = fmaf((float)y * xs, ws, bias);
  asm("" : "+v"(z));
  return z;
}

template <int ODT>
__device__ __forceinline__ void w8_st4(void* out, int64_t i, const float* y) {
  if constexpr (ODT == SL8_DTYPE_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(out) + i) = make_float4(y[0], y[1], y[2], y[3]);
  } else {
    uint32_t z[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = ODT == SL8_DTYPE_F16 ? f2h_bits(y[e]) : f2bf_bits(y[e]);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + i) = make_uint2(z[0] | z[1] << 16, z[2] | z[3] << 16);
  }
}

// ---------------------------------------------------------------------------
// Up to 16 rows: 16 channels at a time, each wave with its part of K: weights straight from memory into A operands
// of v_mfma_i32_16x16x64_i8 (lane (g4, col): 16 bytes of row col), the codes as B operands. The waves' sums
// meet in LDS. Bound by the weights' bytes where a workgroup has many groups of channels (128256 x 4096: 5.4 TB/s;
// 17408 x 5120 in 4.25 rounds, 3.5 to 4). The codes of a wave's part stay in registers while the workgroup goes through
// its groups, a group's weights on their way while the one before is multiplied (behind the last group it reads that one
// again); the two halves of a line are read next to each other (U units of 128 bytes a wave).
// ---------------------------------------------------------------------------
constexpr int W8_WAVES = 8;

// The sums y of channels n .. n + 3 of a row to its outputs.
template <int ODT>
__device__ __forceinline__ void w8_out4(const W8Args& p, v4i y, float xs, int m, int n) {
  float z[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) z[e] = w8_value(y[e], xs, p.ws[min(n + e, p.N - 1)], w8_bias(p, min(n + e, p.N - 1)));
  const int64_t to = (int64_t)m * p.N + n;
  if (p.N % 4 == 0) {
    w8_st4<ODT>(p.out, to, z);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.N) st_out<ODT>(p.out, to + e, z[e]);
  }
}

// XDT 0, 1: x itself, a few fp16 / bf16 rows, is quantised in every workgroup (a launch less; each reads all of x).
constexpr int W8_CODES = -1, W8_FUSED_ROWS = 4;
template <int ODT, int U, int XDT>
__global__ void __launch_bounds__(64 * W8_WAVES) w8_stream_kernel(const W8Args p) {
  constexpr bool FUSED = XDT != W8_CODES;
  __shared__ v4i sum_s[2][W8_WAVES][64];
  __shared__ float amax_s[FUSED ? W8_WAVES : 1][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g4 = lane >> 4;
  const int groups = (p.N + 15) / 16, units = p.Kp / 128;
  const int u0 = wave * units / W8_WAVES, u1 = (wave + 1) * units / W8_WAVES;
  auto load = [&](int64_t g, v4i (&a)[U][2]) __attribute__((always_inline)) {
    const int8_t* w = p.w + (int64_t)min(16 * (int)min(g, (int64_t)groups - 1) + col, p.N - 1) * p.K;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        a[u][i] = *reinterpret_cast<const v4i_u*>(w + min(128 * min(u0 + u, units - 1) + 64 * i + 16 * g4, p.K - 16));
  };
  v4i a0[U][2], a1[U][2], b[U][2];
  float xs = 0.f;  // FUSED: the scale of row lane / 4, which this lane puts out
  // (rows past the last as the last; units past the wave's own are zeros)
  if constexpr (FUSED) {
    uint2 raw[U][2][4];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) w8_raw(p, min(col, p.M - 1), u0 + u < u1 ? 8 * (u0 + u) + 4 * i + g4 : p.Kp / 16, raw[u][i]);
    load(blockIdx.x, a0);
    auto values = [&](const uint2 (&r)[4], float* f) __attribute__((always_inline)) {
      VecIO<XDT>::unpack(make_uint4(r[0].x, r[0].y, r[1].x, r[1].y), f);
      VecIO<XDT>::unpack(make_uint4(r[2].x, r[2].y, r[3].x, r[3].y), f + 8);
    };
    float amax = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float f[16];
        values(raw[u][i], f);
#pragma unroll
        for (int e = 0; e < 16; ++e) amax = w8_top(amax, f[e]);
      }
    amax = w8_top(amax, __shfl_xor(amax, 16, 64));
    amax = w8_top(amax, __shfl_xor(amax, 32, 64));
    if (g4 == 0) amax_s[wave][col] = amax;
    w8_barrier<63>();
    float mine = 0.f;
#pragma unroll
    for (int x = 0; x < W8_WAVES; ++x) {
      amax = w8_top(amax, amax_s[x][col]);
      mine = w8_top(mine, amax_s[x][lane >> 2]);
    }
    auto scale = [](float a) { return a * (1.0f / 127.0f) == 0.f ? 1.f : a * (1.0f / 127.0f); };
    const float safe = scale(amax);
    xs = scale(mine);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float f[16];
        values(raw[u][i], f);
        const uint2 lo = row_codes8<XDT>(f, safe), hi = row_codes8<XDT>(f + 8, safe);
        b[u][i] = v4i{(int)lo.x, (int)lo.y, (int)hi.x, (int)hi.y};
      }
  } else {
    load(blockIdx.x, a0);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int8_t* x = p.codes + ((int64_t)min(u0 + u, units - 1) * p.M16 + min(col, p.M - 1)) * 128;
        const v4i c = *reinterpret_cast<const v4i*>(x + 64 * i + 16 * g4);
        b[u][i] = u0 + u < u1 ? c : v4i{0, 0, 0, 0};
      }
  }
  int turn = 0;
  auto group = [&](int64_t g, const v4i (&a)[U][2], v4i (&next)[U][2]) __attribute__((always_inline)) {
    load(g + gridDim.x, next);
    __builtin_amdgcn_sched_barrier(0);
    v4i acc = {};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u][i], b[u][i], acc, 0, 0, 0);
    sum_s[turn & 1][wave][lane] = acc;
    w8_barrier<63>();  // (a turn's sums are read in front of the next barrier and written again behind it)
    if (wave == turn % W8_WAVES) {  // by turns
      const int m = lane >> 2, n = 16 * (int)g + 4 * (lane & 3);
      v4i y = {0, 0, 0, 0};
#pragma unroll
      for (int x = 0; x < W8_WAVES; ++x) y += sum_s[turn & 1][x][16 * (lane & 3) + m];
      if (m < p.M && n < p.N) w8_out4<ODT>(p, y, FUSED ? xs : p.xs[m], m, n);
    }
    ++turn;
  };
#pragma unroll 1
  for (int64_t g = blockIdx.x; g < groups; g += 2 * gridDim.x) {
    group(g, a0, a1);
    if (g + gridDim.x < groups) group(g + gridDim.x, a1, a0);
  }
}

// ---------------------------------------------------------------------------
// Many rows: BN x BM output tiles (channels x rows), MW waves along the rows and NW along the channels, each
// with 32 NB x 32 MB of them on v_mfma_i32_32x32x32_i8. Stages of 128 bytes of K (whole lines; with 64 bytes
// 512 x 17408 x 5120 took 100 us, 77 now) go through RING places in LDS by direct copies, RING - 1 ahead of the
// products, one barrier a stage; 16-byte chunks of a row are placed by an xor of the row, so that 16 rows of a read lie in
// different banks. Bound by the matrix pipe's power in large tiles (4096 x 17408 x 5120: it is busy in 54 % of the
// cycles, at 1.55 to 1.6 GHz, as the library's product of that size, 385 us, is), by the copies in tiles of 32 and 64
// rows, whose rings are longer for that.
// ---------------------------------------------------------------------------
template <int BM_, int BN_, int MW_, int NW_, int RING_> struct W8Tile {
  static constexpr int RING = RING_;  // stages in LDS
  static constexpr int BM = BM_, BN = BN_, MW = MW_, NW = NW_, BK = W8_BK, THREADS = 64 * MW_ * NW_;
  static constexpr int MB = BM / MW / 32, NB = BN / NW / 32;  // blocks of a wave
  static constexpr int CPR = BK / 16;                           // 16-byte chunks of a row and stage
  static_assert(BM * CPR % THREADS == 0 && BN * CPR % THREADS == 0, "whole copies");
  __device__ __forceinline__ static int swizzle(int row) { return (row >> 1) & 7; }
};

// Tile t: each XCD (workgroup id modulo 8) has a run of them, 8 rows of tiles at a time.
__device__ __forceinline__ void w8_tile_at(const W8Args& p, int id, int& rt, int& ct) {
  if (id < p.whole) {
    const int xcd = id & 7, per = p.whole >> 3, rem = p.whole & 7;
    id = xcd * per + min(xcd, rem) + (id >> 3);
  }
  const int width = 8 * p.nt_n, group = id / width, in = id - group * width;
  const int rows = min(p.nt_m - 8 * group, 8);
  ct = in / rows;
  rt = 8 * group + in - ct * rows;
}

// The wave's sums as outputs: block by block through LDS, to rows of whole lines.
template <int ODT, typename S>
__device__ __forceinline__ void w8_store(const W8Args& p, const v16i (&acc)[S::NB][S::MB], int m0, int n0, int lane,
                                         int8_t* lds) {
  constexpr int OS = ODT == SL8_DTYPE_F32 ? 4 : 2, ROW = S::NB * 32 * OS, CH = ROW / 16;  // bytes, chunks of a row
  const int l32 = lane & 31, h = lane >> 5;
  const bool vec = p.N % (16 / OS) == 0;
  float ws[S::NB][16], bias[S::NB][16];
#pragma unroll
  for (int nb = 0; nb < S::NB; ++nb)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int n = min(n0 + 32 * nb + 8 * (e >> 2) + 4 * h + (e & 3), p.N - 1);
      ws[nb][e] = p.ws[n];
      bias[nb][e] = w8_bias(p, n);
    }
#pragma unroll
  for (int mb = 0; mb < S::MB; ++mb) {
    const int m = m0 + 32 * mb;
    const float xs = p.xs[min(m + l32, p.M - 1)];
    auto place = [&](int row, int chunk) { return lds + row * ROW + 16 * (chunk ^ (row & (CH - 1))); };
#pragma unroll
    for (int nb = 0; nb < S::NB; ++nb)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = w8_value(acc[nb][mb][4 * q + e], xs, ws[nb][4 * q + e], bias[nb][4 * q + e]);
        const int at = (32 * nb + 8 * q + 4 * h) * OS;  // bytes into the row
        if constexpr (OS == 4) {
          *reinterpret_cast<float4*>(place(l32, at / 16)) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
          uint16_t z[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) z[e] = ODT == SL8_DTYPE_F16 ? f2h_bits(y[e]) : f2bf_bits(y[e]);
          *reinterpret_cast<uint2*>(place(l32, at / 16) + at % 16) =
              make_uint2(z[0] | (uint32_t)z[1] << 16, z[2] | (uint32_t)z[3] << 16);
        }
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
    if (vec) {
#pragma unroll
      for (int i = 0; i < 32 * CH / 64; ++i) {
        const int row = (64 * i + lane) / CH, chunk = lane % CH;
        const int n = n0 + chunk * (16 / OS);
        if (m + row < p.M && n < p.N)
          *reinterpret_cast<uint4*>(static_cast<int8_t*>(p.out) + ((int64_t)(m + row) * p.N + n) * OS) =
              *reinterpret_cast<const uint4*>(place(row, chunk));
      }
    } else {
      constexpr int RN = S::NB * 32;
      for (int i = lane; i < 32 * RN; i += 64) {
        const int row = i / RN, n = i % RN;
        if (m + row >= p.M || n0 + n >= p.N) continue;
        const int8_t* from = place(row, n * OS / 16) + n * OS % 16;
        const int64_t to = (int64_t)(m + row) * p.N + n0 + n;
        if constexpr (OS == 4) static_cast<float*>(p.out)[to] = *reinterpret_cast<const float*>(from);
        else static_cast<uint16_t*>(p.out)[to] = *reinterpret_cast<const uint16_t*>(from);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
  }
}

// WIDE: weight rows are 16-byte aligned and copied 16 bytes a thread; else 4 (which is what K % 4 == 0 allows).
template <int ODT, typename S, bool WIDE>
__global__ void __launch_bounds__(S::THREADS, 2) w8_tile_kernel(const W8Args p) {
  constexpr int ROWB = S::BK, STAGE = (S::BM + S::BN) * ROWB, PER = WIDE ? 1 : 4;
  constexpr int WCOP = PER * S::BN * S::CPR / S::THREADS, XCOP = S::BM * S::CPR / S::THREADS;  // copies a thread
  static_assert((S::RING - 2) * (WCOP + XCOP) < 64, "what the wait can count");
  constexpr int OS = ODT == SL8_DTYPE_F32 ? 4 : 2;
  // one LDS object per stage: a copy into one never aliases reads of another
  __shared__ __attribute__((aligned(16))) int8_t s0[STAGE], s1[STAGE], s2[S::RING > 2 ? STAGE : 16],
      s3[S::RING > 3 ? STAGE : 16];
  static_assert(S::MW * S::NW * 32 * S::NB * 32 * OS <= 2 * STAGE, "the outputs fit two stages");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, h = lane >> 5;
  int id = blockIdx.x, split = 0, parts = 1;
  if (id >= p.whole) {
    const int i = id - p.whole;
    id = p.whole + i / p.splits;
    split = i % p.splits;
    parts = p.splits;
  }
  int rt, ct;
  w8_tile_at(p, id, rt, ct);
  const int m0 = rt * S::BM, n0 = ct * S::BN;
  const int nk = p.Kp / S::BK, k0 = split * nk / parts, k1 = (split + 1) * nk / parts;
  const int mw = wave % S::MW, nw = wave / S::MW;

  // copy i of a thread: 16 (weights, not WIDE: 4) bytes of row P / pieces, place P % pieces of it; weight rows past
  // the last read as zeros, rows of codes as the last
  constexpr int WPR = PER * S::CPR;
  const brsrc_t rw = make_rsrc(p.w + (int64_t)n0 * p.K, (uint32_t)(min(S::BN, p.N - n0) * p.K));
  int woff[WCOP], wch[WCOP], xoff[XCOP];
#pragma unroll
  for (int i = 0; i < WCOP; ++i) {
    const int P = i * S::THREADS + tid, row = P / WPR, piece = P % WPR;
    wch[i] = 16 * ((piece / PER) ^ S::swizzle(row));
    woff[i] = row * p.K + 4 * (piece % PER);
  }
#pragma unroll
  for (int i = 0; i < XCOP; ++i) {
    const int P = i * S::THREADS + tid, row = P / S::CPR;  // (as many weight rows in front: a multiple of 16)
    xoff[i] = min(row, p.M16 - m0 - 1) * 128 + 16 * ((P % S::CPR) ^ S::swizzle(row));
  }
  auto load = [&](int kt, int8_t* to) __attribute__((always_inline)) {
    kt = min(kt, k1 - 1);
    const int k = kt * S::BK;
    const brsrc_t rx = make_rsrc(p.codes + ((int64_t)kt * p.M16 + m0) * 128, (uint32_t)(S::BM * 128));
#pragma unroll
    for (int i = 0; i < WCOP; ++i) {
      const int at = woff[i] + min(k + wch[i], p.K - 16);
      if constexpr (WIDE) buf16_to_lds(rw, to + (i * S::THREADS + wave * 64) * 16, at, 0);
      else buf4_to_lds(rw, to + (i * S::THREADS + wave * 64) * 4, at, 0);
    }
#pragma unroll
    for (int i = 0; i < XCOP; ++i)
      buf16_to_lds(rx, to + S::BN * S::BK + (i * S::THREADS + wave * 64) * 16, xoff[i], 0);
  };

  v16i acc[S::NB][S::MB];
#pragma unroll
  for (int nb = 0; nb < S::NB; ++nb)
#pragma unroll
    for (int mb = 0; mb < S::MB; ++mb) acc[nb][mb] = v16i{};
  const int swz = S::swizzle(l32);
  const int wrow = (nw * S::NB * 32 + l32) * ROWB, xrow = (S::BN + mw * S::MB * 32 + l32) * ROWB;
  auto compute = [&](const int8_t* st) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < S::BK / 32; ++ks) {
      const int c = 16 * ((2 * ks + h) ^ swz);
      v4i a[S::NB], b[S::MB];
#pragma unroll
      for (int nb = 0; nb < S::NB; ++nb) a[nb] = *reinterpret_cast<const v4i*>(st + wrow + c + nb * 32 * ROWB);
#pragma unroll
      for (int mb = 0; mb < S::MB; ++mb) b[mb] = *reinterpret_cast<const v4i*>(st + xrow + c + mb * 32 * ROWB);
#pragma unroll
      for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < S::NB; ++nb)
          acc[nb][mb] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[nb], b[mb], acc[nb][mb], 0, 0, 0);
    }
  };
  // (the place of the stage before is free behind the barrier)
  auto step = [&](int kt, const int8_t* st, int8_t* to) __attribute__((always_inline)) {
    w8_barrier<(S::RING - 2) * (WCOP + XCOP)>();
    load(kt + S::RING - 1, to);
    __builtin_amdgcn_sched_barrier(0);
    compute(st);
  };
  int kt = k0;
  load(k0, s0);
  if constexpr (S::RING > 2) {
    load(k0 + 1, s1);
  }
  if constexpr (S::RING > 3) {
    load(k0 + 2, s2);
  }
#pragma unroll 1
  for (; kt + S::RING <= k1; kt += S::RING) {
    if constexpr (S::RING == 2) {
      step(kt, s0, s1);
      step(kt + 1, s1, s0);
    } else if constexpr (S::RING == 3) {
      step(kt, s0, s2);
      step(kt + 1, s1, s0);
      step(kt + 2, s2, s1);
    } else {
      step(kt, s0, s3);
      step(kt + 1, s1, s0);
      step(kt + 2, s2, s1);
      step(kt + 3, s3, s2);
    }
  }
  if (kt < k1) step(kt, s0, S::RING == 2 ? s1 : S::RING == 3 ? s2 : s3);
  if (S::RING > 2 && kt + 1 < k1) step(kt + 1, s1, s0);
  if (S::RING > 3 && kt + 2 < k1) step(kt + 2, s2, s1);
  w8_barrier<0>();  // (copies past the last stage land where the outputs go)
  if (parts > 1) {
    v4i* to = p.part + (int64_t)(blockIdx.x - p.whole) * S::THREADS * (S::NB * S::MB * 4) + tid;
#pragma unroll
    for (int nb = 0; nb < S::NB; ++nb)
#pragma unroll
      for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          to[((nb * S::MB + mb) * 4 + q) * S::THREADS] = v4i{acc[nb][mb][4 * q], acc[nb][mb][4 * q + 1], acc[nb][mb][4 * q + 2],
                                              acc[nb][mb][4 * q + 3]};
    return;
  }
  constexpr int OUTB = 32 * S::NB * 32 * OS, FIT = STAGE / OUTB;
  int8_t* lds = wave < FIT ? s0 + wave * OUTB : s1 + (wave - FIT) * OUTB;
  w8_store<ODT, S>(p, acc, m0 + mw * S::MB * 32, n0 + nw * S::NB * 32, lane, lds);
}

// The parts of the tiles that were split over K, added up: a workgroup for a block of a wave's, a thread for
// four channels of a row, a row's next to each other.
template <int ODT, typename S>
__global__ void __launch_bounds__(256) w8_join_kernel(const W8Args p) {
  constexpr int BLOCKS = S::MW * S::NW * S::NB * S::MB, TILE = BLOCKS * 256;  // of 32 x 32; v4i of a tile
  const int tile = blockIdx.x / BLOCKS, blk = blockIdx.x % BLOCKS;
  const int wave = blk % (S::MW * S::NW), mb = blk / (S::MW * S::NW) % S::MB, nb = blk / (S::MW * S::NW * S::MB);
  const int l32 = threadIdx.x >> 3, q = threadIdx.x >> 1 & 3, h = threadIdx.x & 1;
  int rt, ct;
  w8_tile_at(p, p.whole + tile, rt, ct);
  const int m = rt * S::BM + (wave % S::MW * S::MB + mb) * 32 + l32;
  const int n = ct * S::BN + (wave / S::MW * S::NB + nb) * 32 + 8 * q + 4 * h;
  if (m >= p.M || n >= p.N) return;
  const v4i* from = p.part + (int64_t)tile * p.splits * TILE + ((nb * S::MB + mb) * 4 + q) * S::THREADS + wave * 64 +
                    32 * h + l32;
  v4i y = {0, 0, 0, 0};
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) y += from[(int64_t)s * TILE];
  w8_out4<ODT>(p, y, p.xs[m], m, n);
}

using Tile256 = W8Tile<256, 256, 2, 4, 2>;
using Tile128 = W8Tile<128, 128, 2, 2, 2>;
using Tile64 = W8Tile<64, 128, 1, 4, 3>;
using Tile32 = W8Tile<32, 128, 1, 4, 4>;

// How a call runs.
struct W8Plan {
  int tile;  // rows of an output tile; 0: streamed
  int nt_m, nt_n, whole, splits;
  size_t code_bytes, bytes;
};

// What takes the least time (us): streaming, or a tile and the parts in which the last round's tiles are cut along K.
// Tiles: rounds of the workgroups that are resident at once, each of as many stages as K has, a stage taking
// one_us where a CU has one workgroup, up to full_us where it has per_cu; a join costs its launch and its
// partial sums. Neither is faster than the weights' bytes; launches and the rows' codes are the constants.
// Both sides, calls on one stream: 1 row, 5120 x 5120 streamed 13.0, tiles of 32 rows 15.0; 17408 x 5120 24.7 and 27.1;
// 16 rows, 4096 x 4096 13.0 and 14.9, 30000 x 4096 36.6 and 34.2. Tiles of 32, 64, 128 and 256 rows: 64 rows,
// 17408 x 5120 42.7, 31.9, 37.9, 48.1; 512 rows, 4096 x 4096 23.3, 20.7, 27.1, 30.7 and 17408 x 5120 125, 90.8, 76.7,
// 74.2; 2048 rows, 4096 x 4096 72.2, 55.6, 49.1, 67.2. Where all tiles come to the weights' bytes those of few rows are
// nearer to them, so rows that half a tile holds do not go to it: N = 128256, K = 4096, 1 row 101, 98.5, 111, 124
// (streamed 96.6), 64 rows 136, 112, 122, 140; 57344 x 8192, 8 rows 92.8, 90.8, 102, 117.
W8Plan w8_plan(int64_t M, int64_t N, int64_t K) {
  struct Shape { int bm, bn, per_cu; double one_us, full_us; };
  static const Shape shapes[] = {{256, 256, 1, 1.7, 1.7}, {128, 128, 2, 0.9, 1.2}, {64, 128, 2, 0.6, 0.95}, {32, 128, 2, 0.45, 0.8}};
  W8Plan a{};
  a.code_bytes = ((size_t)((M + 15) / 16 * 16) * w8_padded(K) + (size_t)M * sizeof(float) + 15) / 16 * 16;
  a.bytes = a.code_bytes;
  a.splits = 1;
  const double stages = (double)w8_padded(K) / W8_BK, cus = cu_count();
  double best = 1e30;
  if (M <= W8_STREAM_ROWS && K <= W8_STREAM_K) best = M <= W8_FUSED_ROWS ? 3.5 + (double)N * K / 4.6e6 : 6. + (double)N * K / 4.2e6;
  for (const Shape& s : shapes) {
    if (s.bm > 32 && 2 * M <= s.bm) continue;  // a tile of half the rows holds them all
    const int64_t nt_m = (M + s.bm - 1) / s.bm, nt_n = (N + s.bn - 1) / s.bn, n = nt_m * nt_n;
    const int64_t slots = (int64_t)cus * s.per_cu, rest = n % slots, most = n - rest;
    for (int S = 1; S <= 8; ++S) {
      if (S > 1 && (rest == 0 || stages < 4 * S || rest * S > slots)) break;
      const double more = std::ceil((double)rest * S / cus) - 1.;
      const double part = rest ? std::ceil(stages / S) * (s.one_us + (s.full_us - s.one_us) * more / std::max(1, s.per_cu - 1)) : 0.;
      double us = std::max((double)(most / slots) * stages * s.full_us + part, (double)N * K / 4.8e6) + 6.;
      if (S > 1) us += 3.5 + (double)rest * S * s.bm * s.bn * 5 / 4e6;
      if (us >= best) continue;
      best = us;
      a.tile = s.bm;
      a.nt_m = (int)nt_m;
      a.nt_n = (int)nt_n;
      a.splits = S;
      a.whole = (int)(S > 1 ? most : n);
      a.bytes = a.code_bytes + (S > 1 ? (size_t)rest * S * s.bm * s.bn * 4 : 0);
    }
  }
  return a;
}

}  // namespace
}  // namespace sl8

using namespace sl8;

extern "C" size_t sl8_linear_w8a8_workspace(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K < 16 || M >= (1LL << 24) || N >= (1LL << 24) || K >= W8_MAX_K) return 0;
  return w8_plan(M, N, K).bytes;
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
  SL8_CHECK_ARG(M >= 0 && N >= 0 && M < (1LL << 24) && N < (1LL << 24), "fni8 %s: shape too large", tag);
  SL8_CHECK_ARG(K >= 16 && K % 4 == 0 && K < W8_MAX_K,
                "fni8 %s: K must be a multiple of 4, 16 to %d, got %lld", tag, W8_MAX_K - 4, (long long)K);
  if (M == 0 || N == 0) return SL8_OK;
  SL8_CHECK_ARG(x && w && w_scale && out, "fni8 %s: null pointer", tag);
  SL8_CHECK_ARG(aligned(w, K % 16 ? 4 : 16), "fni8 %s: w must be 16-byte aligned (4 where K %% 16 != 0)", tag);
  SL8_CHECK_ARG(aligned(x, 16) && aligned(out, 16), "fni8 %s: x/out must be 16-byte aligned", tag);
  const W8Plan plan = w8_plan(M, N, K);
  SL8_CHECK_ARG(workspace && aligned(workspace, 16) && workspace_bytes >= plan.bytes,
                "fni8 %s: workspace needs %zu bytes", tag, plan.bytes);
  W8Args p{};
  p.x = x; p.w = w; p.ws = w_scale; p.bias = bias; p.out = out;
  p.bias_dt = bias ? bias_dtype : -1;
  p.M = (int)M; p.N = (int)N; p.K = (int)K; p.Kp = (int)w8_padded(K); p.M16 = (int)((M + 15) / 16 * 16);
  p.codes = static_cast<int8_t*>(workspace);
  p.xs = reinterpret_cast<float*>(p.codes + (int64_t)p.M16 * p.Kp);
  p.part = reinterpret_cast<v4i*>(p.codes + plan.code_bytes);
  p.nt_m = plan.nt_m; p.nt_n = plan.nt_n; p.whole = plan.whole; p.splits = plan.splits;
  const int64_t split = (int64_t)plan.nt_m * plan.nt_n - plan.whole, grid = plan.whole + split * plan.splits;
  SL8_CHECK_ARG(grid < (1LL << 32) / 512 && M < (1LL << 32) / 256, "fni8 %s: shape too large", tag);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  using std::integral_constant;
  auto quant = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (p.Kp <= 4096) w8_quant_kernel<DT, 1><<<(unsigned)M, 256, 0, st>>>(p);
    else if (p.Kp <= 8192) w8_quant_kernel<DT, 2><<<(unsigned)M, 256, 0, st>>>(p);
    else if (p.Kp <= 16384) w8_quant_kernel<DT, 4><<<(unsigned)M, 256, 0, st>>>(p);
    else w8_quant_kernel<DT, 0><<<(unsigned)M, 256, 0, st>>>(p);
  };
  // up to W8_FUSED_ROWS 16-bit rows that are streamed: no launch for their codes
  const bool fused = plan.tile == 0 && M <= W8_FUSED_ROWS && x_dtype != SL8_DTYPE_F32;
  if (fused) {
  } else if (x_dtype == SL8_DTYPE_F16) quant(integral_constant<int, SL8_DTYPE_F16>{});
  else if (x_dtype == SL8_DTYPE_BF16) quant(integral_constant<int, SL8_DTYPE_BF16>{});
  else quant(integral_constant<int, SL8_DTYPE_F32>{});
  auto go = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (plan.tile == 0) {
      // (as many as are resident: a wave's codes and two groups of weights take up to 245 registers. With twice as
      // many 5120 x 5120 takes 18.4 for 13.0 us)
      const unsigned wgs = (unsigned)std::min<int64_t>((N + 15) / 16, (int64_t)cu_count() * (K <= 2048 ? 2 : 1));
      auto stream = [&](auto xdt) {
        constexpr int XDT = decltype(xdt)::value;
        if (K <= 2048) w8_stream_kernel<DT, 2, XDT><<<wgs, 64 * W8_WAVES, 0, st>>>(p);
        else if (K <= 4096) w8_stream_kernel<DT, 4, XDT><<<wgs, 64 * W8_WAVES, 0, st>>>(p);
        else w8_stream_kernel<DT, 5, XDT><<<wgs, 64 * W8_WAVES, 0, st>>>(p);
      };
      if (!fused) stream(integral_constant<int, W8_CODES>{});
      else if (x_dtype == SL8_DTYPE_F16) stream(integral_constant<int, SL8_DTYPE_F16>{});
      else stream(integral_constant<int, SL8_DTYPE_BF16>{});
      return;
    }
    auto tile = [&](auto shape) {
      using S = decltype(shape);
      if (K % 16 == 0) w8_tile_kernel<DT, S, true><<<(unsigned)grid, S::THREADS, 0, st>>>(p);
      else w8_tile_kernel<DT, S, false><<<(unsigned)grid, S::THREADS, 0, st>>>(p);
      if (split) w8_join_kernel<DT, S><<<(unsigned)(split * (S::BM * S::BN / 1024)), 256, 0, st>>>(p);
    };
    if (plan.tile == 256) tile(Tile256{});
    else if (plan.tile == 128) tile(Tile128{});
    else if (plan.tile == 64) tile(Tile64{});
    else tile(Tile32{});
  };
  if (out_dtype == SL8_DTYPE_F16) go(integral_constant<int, SL8_DTYPE_F16>{});
  else if (out_dtype == SL8_DTYPE_BF16) go(integral_constant<int, SL8_DTYPE_BF16>{});
  else go(integral_constant<int, SL8_DTYPE_F32>{});
  SL8_CHECK_LAUNCH(tag);
  return SL8_OK;
}
