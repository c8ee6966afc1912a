// Rotary positions: the angles of a token's pairs and the turned rows, for the rotation of its own
// (rope.hip) and the one on the way into a paged cache (block8.hip).
//
// Pair p of a row of D elements, R of them rotary, is (x_i, x_j) with (i, j) = (p, p + R/2), or
// (2p, 2p + 1) interleaved; it turns by the angle of its axis' position:
//   x_i' = x_i cos - x_j sin,  x_j' = x_j cos + x_i sin,
// cos = table[pos][p], sin = table[pos][R/2 + p] (fp32, made by the caller in any way: far
// positions keep their angles, which 32-bit products of position and frequency would not). The
// inverse (the transpose, hence the gradient) takes -sin. Elements R..D-1 pass.
#pragma once

#include "common.hpp"
#include "rowquant.hpp"

namespace sl8 {
namespace {

constexpr int ROPE_MAX_AXES = 4;

struct RopeArgs {
  const void* pos;    // [axes][tokens] or, with pos_b = 0, [axes][S]; int32 or int64
  int64_t pos_axis;   // elements between axes
  int64_t pos_b;      // elements between the sequences of a batch (0: shared)
  const float* table;
  int64_t rows;       // positions of the table; others are taken as its nearest end
  int R;
  int end[ROPE_MAX_AXES];  // first pair past each axis; unused axes R / 2
  int axes;
  bool pos64, interleaved, inverse;

  __device__ __forceinline__ int64_t at(int axis, int64_t token) const {
    const int64_t i = axis * pos_axis + token;
    const int64_t p = pos64 ? static_cast<const int64_t*>(pos)[i] : static_cast<const int32_t*>(pos)[i];
    return p < 0 ? 0 : p < rows ? p : rows - 1;
  }
  __device__ __forceinline__ int axis_of(int pair) const {
    return (pair >= end[0]) + (pair >= end[1]) + (pair >= end[2]);
  }
};

template <int N>
__device__ __forceinline__ void ld_f32(const float* p, float* f) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) VecIO<SL8_DTYPE_F32>::unpack(*reinterpret_cast<const uint4*>(p + i), f + i);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = p[i];
  }
}

// cos and sin of pairs p0 .. p0 + N - 1 (N = 4, 8: p0, R / 2 and the table aligned to 4 floats)
// of a token; sin negated for the inverse. Where a thread's pairs belong to several axes, each
// takes a position and two angles of its own: 4 x 4096 tokens, 16 + 16 heads, D = 80, fp16, two axes of
// 20 pairs 49 us, one axis 40; 6121 tokens, bf16, axes of (15, 25, 24) pairs 25.9, of (16, 24, 24), which
// no thread's 8 straddle, 22.7.
template <int N>
__device__ __forceinline__ void rope_angles(const RopeArgs& a, int64_t token, int p0, float* c, float* s) {
  const int half = a.R / 2;
  const int ax = a.axis_of(p0);
  if (a.axes == 1 || ax == a.axis_of(p0 + N - 1)) {
    const float* row = a.table + a.at(ax, token) * a.R;
    ld_f32<N>(row + p0, c);
    ld_f32<N>(row + half + p0, s);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float* row = a.table + a.at(a.axis_of(p0 + e), token) * a.R;
      c[e] = row[p0 + e];
      s[e] = row[half + p0 + e];
    }
  }
  if (a.inverse) {
#pragma unroll
    for (int e = 0; e < N; ++e) s[e] = -s[e];
  }
}

// N consecutive elements of a row as fp32 and back.
template <int DT, int N>
__device__ __forceinline__ void ld_elems(const void* base, int64_t i, float* f) {
  using T = typename Elem<DT>::T;
  const T* p = static_cast<const T*>(base) + i;
  if constexpr (DT == SL8_DTYPE_F32) {
    ld_f32<N>(p, f);
  } else if constexpr (N == 8) {
    VecIO<DT>::unpack(*reinterpret_cast<const uint4*>(p), f);
  } else if constexpr (N == 4) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    f[0] = u16_to_f<DT>(v.x & 0xFFFF); f[1] = u16_to_f<DT>(v.x >> 16);
    f[2] = u16_to_f<DT>(v.y & 0xFFFF); f[3] = u16_to_f<DT>(v.y >> 16);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = Elem<DT>::ld(p, e);
  }
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == SL8_DTYPE_F16) return (uint32_t)f2h_bits(a) | ((uint32_t)f2h_bits(b) << 16);
  else return (uint32_t)f2bf_bits(a) | ((uint32_t)f2bf_bits(b) << 16);
}
template <int DT, int N>
__device__ __forceinline__ void st_elems(void* base, int64_t i, const float* f) {
  if constexpr (DT == SL8_DTYPE_F32) {
    float* p = static_cast<float*>(base) + i;
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int e = 0; e < N; e += 4) *reinterpret_cast<float4*>(p + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) p[e] = f[e];
    }
  } else {
    uint16_t* p = static_cast<uint16_t*>(base) + i;
    if constexpr (N == 8)
      *reinterpret_cast<uint4*>(p) = make_uint4(pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]),
                                                pack2<DT>(f[4], f[5]), pack2<DT>(f[6], f[7]));
    else if constexpr (N == 4)
      *reinterpret_cast<uint2*>(p) = make_uint2(pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]));
    else
#pragma unroll
      for (int e = 0; e < N; ++e) st_out<DT>(base, i + e, f[e]);
  }
}

// Rows of Q and K [B, H, S, D] in any strides (elements; the last dimension dense), in and out. A
// thread holds 2 N elements of a row: N pairs, or 2 N that pass; D / (2 N) threads a row. It keeps
// its pairs' angles for the heads that it visits: the angles are 2 R / D times an fp16 row's
// bytes. A workgroup has `tokens` tokens by `slots` head slots.
struct RopeRows {
  const void *q, *k;
  void *q_out, *k_out;
  int64_t qs[3], ks[3], qo[3], ko[3];  // strides of b, h, s
  int64_t T, S;          // B * S rows a head
  int Hq, Hkv, D;
  int slots, tokens;
};

template <int DT, int N>
__device__ __forceinline__ void rope_block(const RopeArgs& a, const RopeRows& t, int64_t block) {
  const int ch = t.D / (2 * N);
  const int row = threadIdx.x / ch, c = threadIdx.x % ch;
  if (row >= t.slots * t.tokens) return;
  const int64_t tok = block * t.tokens + row / t.slots;
  if (tok >= t.T) return;
  const int64_t b = tok / t.S, s = tok % t.S;
  const int half = a.R / 2;
  const bool turn = c * N < half;
  float co[N], si[N];
  int i0, j0;
  if (turn) {
    rope_angles<N>(a, b * a.pos_b + s, c * N, co, si);
    i0 = a.interleaved ? 2 * N * c : N * c;
    j0 = a.interleaved ? i0 + N : i0 + half;
  } else {
    i0 = 2 * N * c;
    j0 = i0 + N;
  }
  const int H = t.Hq + t.Hkv;
  for (int h = row % t.slots; h < H; h += t.slots) {
    const bool isk = h >= t.Hq;
    const int hh = isk ? h - t.Hq : h;
    const void* x = isk ? t.k : t.q;
    const int64_t in = b * (isk ? t.ks[0] : t.qs[0]) + hh * (isk ? t.ks[1] : t.qs[1]) +
                       s * (isk ? t.ks[2] : t.qs[2]);
    const int64_t to = b * (isk ? t.ko[0] : t.qo[0]) + hh * (isk ? t.ko[1] : t.qo[1]) +
                       s * (isk ? t.ko[2] : t.qo[2]);
    float f[2 * N];
    ld_elems<DT, N>(x, in + i0, f);
    ld_elems<DT, N>(x, in + j0, f + N);
    if (turn) {
      if (a.interleaved) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float u = f[2 * e], v = f[2 * e + 1];
          f[2 * e] = u * co[e] - v * si[e];
          f[2 * e + 1] = v * co[e] + u * si[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float u = f[e], v = f[N + e];
          f[e] = u * co[e] - v * si[e];
          f[N + e] = v * co[e] + u * si[e];
        }
      }
    }
    void* y = isk ? t.k_out : t.q_out;
    st_elems<DT, N>(y, to + i0, f);
    st_elems<DT, N>(y, to + j0, f + N);
  }
}

// Pairs a thread may hold: what divides the row and what the addresses are aligned to.
inline int rope_pairs(int64_t D, int64_t R, int dtype, const void* const* ptrs, int np,
                      const int64_t* strides, int ns) {
  const int64_t size = dtype == SL8_DTYPE_F32 ? 4 : 2;
  for (int n = 16 / (int)size; n >= 4; n /= 2) {  // (16-byte accesses next to each other, or 8)
    const int64_t bytes = n * size;
    bool ok = D % (2 * n) == 0 && R % (2 * n) == 0;
    for (int i = 0; i < np; ++i) ok = ok && aligned(ptrs[i], (uintptr_t)bytes);
    for (int i = 0; i < ns; ++i) ok = ok && strides[i] * size % bytes == 0;
    if (ok) return n;
  }
  return 1;
}

// Head slots and tokens of a workgroup: passes over the heads that leave the fewest of its
// `rows` rows without one.
inline void rope_shape(RopeRows& t, int rows) {
  const int H = t.Hq + t.Hkv;
  double best = 0;
  for (int n = 1; n <= 8 && n <= H; ++n) {
    const int slots = (H + n - 1) / n;
    if (slots > rows) continue;
    const int tokens = rows / slots;
    const double use = (double)tokens * H / ((double)rows * n);
    if (use > best) {
      best = use;
      t.slots = slots;
      t.tokens = tokens;
    }
  }
  if (best == 0) {  // more than 8 * rows heads
    t.slots = rows;
    t.tokens = 1;
  }
}

// The checks shared by the entry points that rotate; fills `a`.
inline int rope_args(const char* tag, RopeArgs& a, const void* pos, int pos64, int64_t pos_axis,
                     int64_t pos_b, const float* table, int64_t rows, int64_t R, int64_t D,
                     const int32_t* sections, int axes, int interleaved, int inverse) {
  SL8_CHECK_ARG(R >= 2 && R % 2 == 0 && R <= D, "fni8 %s: rotary dim must be even and at most the head dim, got %lld",
                tag, (long long)R);
  SL8_CHECK_ARG(axes >= 1 && axes <= ROPE_MAX_AXES, "fni8 %s: 1..%d position axes, got %d", tag,
                ROPE_MAX_AXES, axes);
  SL8_CHECK_ARG(rows >= 1, "fni8 %s: the table has no positions", tag);
  SL8_CHECK_ARG(pos && table, "fni8 %s: null pointer", tag);
  SL8_CHECK_ARG(aligned(table, 16) && aligned(pos, pos64 ? 8 : 4), "fni8 %s: table must be 16-byte aligned", tag);
  a = RopeArgs{pos, pos_axis, pos_b, table, rows, (int)R, {}, axes, pos64 != 0, interleaved != 0, inverse != 0};
  int64_t p = 0;
  for (int i = 0; i < ROPE_MAX_AXES; ++i) {
    if (axes > 1 && i < axes) {
      SL8_CHECK_ARG(sections && sections[i] > 0, "fni8 %s: sections must be positive", tag);
      p += sections[i];
    } else {
      p = R / 2;
    }
    a.end[i] = (int)p;
    if (axes > 1 && i == axes - 1)
      SL8_CHECK_ARG(p == R / 2, "fni8 %s: sections must add up to half the rotary dim", tag);
  }
  return SL8_OK;
}

}  // namespace
}  // namespace sl8
