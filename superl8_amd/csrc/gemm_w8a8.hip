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
constexpr int W8_BK = 64;      // bytes of K a stage of the tile kernel, and what a row's codes are padded to
constexpr int W8_STREAM = 64;  // most rows of x that stream the weights

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
  v4i* part;  // sums of the tiles that are split over K
  int M, N, K, Kp;
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
    for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(x[e]));
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
  amax = fmaxf(fmaxf(amax_s[0], amax_s[1]), fmaxf(amax_s[2], amax_s[3]));
  const float s = amax * (1.0f / 127.0f), safe = s == 0.f ? 1.f : s;
  if (threadIdx.x == 0) p.xs[row] = safe;
  auto put = [&](int c, const float* x) {
    const uint2 lo = row_codes8<DT>(x, safe), hi = row_codes8<DT>(x + 8, safe);
    if (c < chunks) *reinterpret_cast<uint4*>(p.codes + row * p.Kp + 16 * c) = make_uint4(lo.x, lo.y, hi.x, hi.y);
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

typedef v4i v4i_u __attribute__((aligned(4)));  // rows of K % 16 != 0 are 4-byte aligned

__device__ __forceinline__ float w8_bias(const W8Args& p, int n) {
  if (p.bias_dt < 0) return 0.f;
  if (p.bias_dt == SL8_DTYPE_F32) return static_cast<const float*>(p.bias)[n];
  const uint16_t b = static_cast<const uint16_t*>(p.bias)[n];
  return p.bias_dt == SL8_DTYPE_F16 ? h2f(b) : bf2f(b);
}

// ---------------------------------------------------------------------------
// Few rows: each wave streams 16 NR weight rows' part of K straight into A operands of
// v_mfma_i32_16x16x64_i8 (lane (g4, col): 16 bytes of row col), x's codes are the B operands; the 8 waves of a
// workgroup have an eighth of K each and add their sums in LDS. Bound by the weights' bytes.
// ---------------------------------------------------------------------------
constexpr int WS_WAVES = 8;

template <int ODT, int RT, int NR>
__global__ void __launch_bounds__(64 * WS_WAVES) w8_stream_kernel(const W8Args p) {
  constexpr int U = NR * RT <= 2 ? 4 : 2;  // steps whose loads go out together
  __shared__ v4i sum_s[WS_WAVES][NR * RT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g4 = lane >> 4;
  const int n0 = blockIdx.x * 16 * NR;
  const int8_t *w[NR], *x[RT];
#pragma unroll
  for (int r = 0; r < NR; ++r) w[r] = p.w + (int64_t)min(n0 + 16 * r + col, p.N - 1) * p.K;
#pragma unroll
  for (int r = 0; r < RT; ++r) x[r] = p.codes + (int64_t)min(16 * r + col, p.M - 1) * p.Kp;
  v4i acc[NR][RT] = {};
  const int steps = p.Kp / 64, s0 = wave * steps / WS_WAVES, s1 = (wave + 1) * steps / WS_WAVES;
  for (int s = s0; s < s1; s += U) {
    v4i a[U][NR], b[U][RT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = 64 * min(s + u, s1 - 1) + 16 * g4;
#pragma unroll
      for (int r = 0; r < NR; ++r) a[u][r] = *reinterpret_cast<const v4i_u*>(w[r] + min(k, p.K - 16));
#pragma unroll
      for (int r = 0; r < RT; ++r) b[u][r] = *reinterpret_cast<const v4i*>(x[r] + k);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u >= s1) break;
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int t = 0; t < RT; ++t)
          acc[r][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u][r], b[u][t], acc[r][t], 0, 0, 0);
    }
  }
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int t = 0; t < RT; ++t) sum_s[wave][r * RT + t][lane] = acc[r][t];
  __syncthreads();
  for (int i = threadIdx.x; i < NR * RT * 64; i += 64 * WS_WAVES) {
    const int blk = i >> 6, l = i & 63, m = 16 * (blk % RT) + (l & 15), n = n0 + 16 * (blk / RT) + 4 * (l >> 4);
    v4i y = {0, 0, 0, 0};
#pragma unroll
    for (int x2 = 0; x2 < WS_WAVES; ++x2) y += sum_s[x2][blk][l];
    if (m >= p.M) continue;
    const float xs = p.xs[m];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.N) st_out<ODT>(p.out, (int64_t)m * p.N + n + e, (float)y[e] * xs * p.ws[n + e] + w8_bias(p, n + e));
  }
}

// ---------------------------------------------------------------------------
// Many rows: BN x BM output tiles (channels x rows), MW waves along the rows and NW along the channels, each
// with 32 NB x 32 MB of them on v_mfma_i32_32x32x32_i8. Stages of 64 bytes of K go through a ring of four in
// LDS by direct copies, three stages ahead; 16-byte chunks of a row are placed by an xor of the row, so that
// 16 rows of a read lie in different banks.
// ---------------------------------------------------------------------------
template <int BM_, int BN_, int MW_, int NW_> struct W8Tile {
  static constexpr int BM = BM_, BN = BN_, MW = MW_, NW = NW_, THREADS = 64 * MW_ * NW_;
  static constexpr int MB = BM / MW / 32, NB = BN / NW / 32;  // blocks of a wave
  static constexpr int COPIES = (BM + BN) * 4 / THREADS;      // of 16 bytes a thread and stage
  static_assert((BM + BN) * 4 % THREADS == 0 && BN * 4 % THREADS == 0, "whole copies");
};

// A barrier behind which the workgroup's copies have arrived but for the last N of each thread, and the reads
// in front of it are done. (A fence would wait for all copies.)
template <int N> __device__ __forceinline__ void w8_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);  // vmcnt(N) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

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
        for (int e = 0; e < 4; ++e) y[e] = (float)acc[nb][mb][4 * q + e] * xs * ws[nb][4 * q + e] + bias[nb][4 * q + e];
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

// DMA: 16-byte aligned weight rows, copied straight to LDS; else through registers.
template <int ODT, typename S, bool DMA>
__global__ void __launch_bounds__(S::THREADS, 2) w8_tile_kernel(const W8Args p) {
  constexpr int ROWB = W8_BK, STAGE = (S::BM + S::BN) * ROWB, WCOP = S::BN * 4 / S::THREADS;
  constexpr int OS = ODT == SL8_DTYPE_F32 ? 4 : 2;
  // one LDS object per stage: a copy into one never aliases reads of another
  __shared__ __attribute__((aligned(16))) int8_t s0[STAGE], s1[STAGE], s2[STAGE], s3[STAGE];
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
  const int nk = p.Kp / W8_BK, k0 = split * nk / parts, k1 = (split + 1) * nk / parts;
  const int mw = wave % S::MW, nw = wave / S::MW;

  // chunk P of a stage: row P / 4 (weights, then x), place P % 4 of it
  const brsrc_t rw = make_rsrc(p.w + (int64_t)n0 * p.K, (uint32_t)(min(S::BN, p.N - n0) * p.K));
  const brsrc_t rx = make_rsrc(p.codes + (int64_t)m0 * p.Kp, (uint32_t)(min(S::BM, p.M - m0) * p.Kp));
  int off[S::COPIES], ch[S::COPIES];
#pragma unroll
  for (int i = 0; i < S::COPIES; ++i) {
    const int P = i * S::THREADS + tid, row = P / 4;
    ch[i] = 16 * ((P & 3) ^ ((row >> 2) & 3));
    if (i < WCOP) off[i] = min(row, p.N - n0 - 1) * p.K;
    else off[i] = min(row - S::BN, p.M - m0 - 1) * p.Kp;
  }
  v4i held[DMA ? 1 : S::COPIES];
  auto load = [&](int kt, int8_t* to) __attribute__((always_inline)) {
    const int k = min(kt, k1 - 1) * W8_BK;
#pragma unroll
    for (int i = 0; i < S::COPIES; ++i) {
      const bool is_w = i < WCOP;
      const int at = is_w ? off[i] + min(k + ch[i], p.K - 16) : off[i] + k + ch[i];
      if constexpr (DMA) buf16_to_lds(is_w ? rw : rx, to + (i * S::THREADS + wave * 64) * 16, at, 0);
      else if (is_w) held[i] = *reinterpret_cast<const v4i_u*>(p.w + (int64_t)n0 * p.K + at);
      else held[i] = *reinterpret_cast<const v4i*>(p.codes + (int64_t)m0 * p.Kp + at);
    }
  };
  auto keep = [&](int8_t* to) __attribute__((always_inline)) {
    if constexpr (!DMA) {
#pragma unroll
      for (int i = 0; i < S::COPIES; ++i) *reinterpret_cast<v4i*>(to + (i * S::THREADS + tid) * 16) = held[i];
    }
  };

  v16i acc[S::NB][S::MB];
#pragma unroll
  for (int nb = 0; nb < S::NB; ++nb)
#pragma unroll
    for (int mb = 0; mb < S::MB; ++mb) acc[nb][mb] = v16i{};
  const int swz = (l32 >> 2) & 3;
  const int wrow = (nw * S::NB * 32 + l32) * ROWB, xrow = (S::BN + mw * S::MB * 32 + l32) * ROWB;
  auto compute = [&](const int8_t* st) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
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
  // stage kt is there when all but the copies of the two behind it have arrived; the ring's place of the stage
  // before it is free behind the barrier
  auto step = [&](int kt, const int8_t* st, int8_t* to) __attribute__((always_inline)) {
    w8_barrier<DMA ? 2 * S::COPIES : 63>();
    load(kt + 3, to);
    compute(st);
    keep(to);
  };
  load(k0, s0);
  keep(s0);
  load(k0 + 1, s1);
  keep(s1);
  load(k0 + 2, s2);
  keep(s2);
  int kt = k0;
#pragma unroll 1
  for (; kt + 4 <= k1; kt += 4) {
    step(kt, s0, s3);
    step(kt + 1, s1, s0);
    step(kt + 2, s2, s1);
    step(kt + 3, s3, s2);
  }
  if (kt < k1) step(kt, s0, s3);
  if (kt + 1 < k1) step(kt + 1, s1, s0);
  if (kt + 2 < k1) step(kt + 2, s2, s1);
  w8_barrier<0>();  // (copies past the last stage land where the outputs go)
  if (parts > 1) {
    v4i* to = p.part + ((int64_t)(blockIdx.x - p.whole) * S::THREADS + tid) * (S::NB * S::MB * 4);
#pragma unroll
    for (int nb = 0; nb < S::NB; ++nb)
#pragma unroll
      for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          to[(nb * S::MB + mb) * 4 + q] = v4i{acc[nb][mb][4 * q], acc[nb][mb][4 * q + 1], acc[nb][mb][4 * q + 2],
                                              acc[nb][mb][4 * q + 3]};
    return;
  }
  constexpr int OUTB = 32 * S::NB * 32 * OS, FIT = STAGE / OUTB;
  int8_t* lds = wave < FIT ? s0 + wave * OUTB : s1 + (wave - FIT) * OUTB;
  w8_store<ODT, S>(p, acc, m0 + mw * S::MB * 32, n0 + nw * S::NB * 32, lane, lds);
}

// The parts of a tile that was split over K, added up.
template <int ODT, typename S>
__global__ void __launch_bounds__(S::THREADS) w8_join_kernel(const W8Args p) {
  constexpr int OS = ODT == SL8_DTYPE_F32 ? 4 : 2, OUTB = 32 * S::NB * 32 * OS;
  __shared__ __attribute__((aligned(16))) int8_t lds[S::MW * S::NW * OUTB];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int rt, ct;
  w8_tile_at(p, p.whole + blockIdx.x, rt, ct);
  v16i acc[S::NB][S::MB];
#pragma unroll
  for (int nb = 0; nb < S::NB; ++nb)
#pragma unroll
    for (int mb = 0; mb < S::MB; ++mb) acc[nb][mb] = v16i{};
  for (int s = 0; s < p.splits; ++s) {
    const v4i* from = p.part + ((int64_t)(blockIdx.x * p.splits + s) * S::THREADS + tid) * (S::NB * S::MB * 4);
#pragma unroll
    for (int nb = 0; nb < S::NB; ++nb)
#pragma unroll
      for (int mb = 0; mb < S::MB; ++mb)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const v4i y = from[(nb * S::MB + mb) * 4 + q];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[nb][mb][4 * q + e] += y[e];
        }
  }
  w8_store<ODT, S>(p, acc, rt * S::BM + wave % S::MW * S::MB * 32, ct * S::BN + wave / S::MW * S::NB * 32, lane,
                   lds + wave * OUTB);
}

using Tile256 = W8Tile<256, 256, 2, 4>;
using Tile128 = W8Tile<128, 128, 2, 2>;

// How a call runs.
struct W8Plan {
  int rows;  // streamed: rows of x in steps of 16; 0: tiles
  bool big;
  int nt_m, nt_n, whole, splits;
  size_t code_bytes, bytes;
};

W8Plan w8_plan(int64_t M, int64_t N, int64_t K) {
  W8Plan a{};
  a.code_bytes = ((size_t)M * (w8_padded(K) + sizeof(float)) + 15) / 16 * 16;
  a.bytes = a.code_bytes;
  a.splits = 1;
  if (M <= W8_STREAM) {
    a.rows = (int)((M + 15) / 16);
    return a;
  }
  const int64_t cus = cu_count();
  auto tiles = [&](int64_t b) { return ((M + b - 1) / b) * ((N + b - 1) / b); };
  a.big = tiles(256) >= cus;
  const int64_t b = a.big ? 256 : 128, n = tiles(b), slots = a.big ? cus : 2 * cus;
  a.nt_m = (int)((M + b - 1) / b);
  a.nt_n = (int)((N + b - 1) / b);
  const int64_t rest = n % slots;
  a.whole = (int)n;
  if (rest && rest * 2 <= slots && K >= 1024) {
    a.splits = (int)std::min<int64_t>(std::min<int64_t>(slots / rest, K / 512), 8);
    a.whole = (int)(n - rest);
    a.bytes += (size_t)rest * a.splits * b * b * 4;
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
  p.M = (int)M; p.N = (int)N; p.K = (int)K; p.Kp = (int)w8_padded(K);
  p.codes = static_cast<int8_t*>(workspace);
  p.xs = reinterpret_cast<float*>(p.codes + M * p.Kp);
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
  if (x_dtype == SL8_DTYPE_F16) quant(integral_constant<int, SL8_DTYPE_F16>{});
  else if (x_dtype == SL8_DTYPE_BF16) quant(integral_constant<int, SL8_DTYPE_BF16>{});
  else quant(integral_constant<int, SL8_DTYPE_F32>{});
  auto go = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (plan.rows) {
      constexpr int NR = 2;
      const unsigned wgs = (unsigned)((N + 16 * NR - 1) / (16 * NR));
      if (plan.rows == 1) w8_stream_kernel<DT, 1, NR><<<wgs, 64 * WS_WAVES, 0, st>>>(p);
      else if (plan.rows == 2) w8_stream_kernel<DT, 2, NR><<<wgs, 64 * WS_WAVES, 0, st>>>(p);
      else w8_stream_kernel<DT, 4, NR><<<wgs, 64 * WS_WAVES, 0, st>>>(p);
      return;
    }
    auto tile = [&](auto shape) {
      using S = decltype(shape);
      if (K % 16 == 0) w8_tile_kernel<DT, S, true><<<(unsigned)grid, S::THREADS, 0, st>>>(p);
      else w8_tile_kernel<DT, S, false><<<(unsigned)grid, S::THREADS, 0, st>>>(p);
      if (split) w8_join_kernel<DT, S><<<(unsigned)split, S::THREADS, 0, st>>>(p);
    };
    if (plan.big) tile(Tile256{});
    else tile(Tile128{});
  };
  if (out_dtype == SL8_DTYPE_F16) go(integral_constant<int, SL8_DTYPE_F16>{});
  else if (out_dtype == SL8_DTYPE_BF16) go(integral_constant<int, SL8_DTYPE_BF16>{});
  else go(integral_constant<int, SL8_DTYPE_F32>{});
  SL8_CHECK_LAUNCH(tag);
  return SL8_OK;
}
