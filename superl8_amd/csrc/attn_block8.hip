// Attention of new tokens over the block-scaled paged int8 cache (block8.hpp). No counterpart in
// the reference, whose paged cache has a scale per token and one query token per sequence.
//
// Query row i of a sequence's n new ones stands at position p = len - n + i and sees keys j <= p,
// with a window j > p - window too. Its row (rotated by the Hadamard matrix as the keys were, in
// 32 bits) is quantised to int8 with one scale qs; then
//   s_j = qs * scale * log2(e) * ks[block(j)] * <q, k_j> (exact integers inside),
//   out = sum_j 2^s_j vs[block(j)] v_j / sum_j 2^s_j;
// a row that sees nothing gives zeros. The scale of V goes into the exponent: with
//   t_j = s_j + log2 vs, m near max t_j, w_j = 2^(t_j - m):  out = sum w_j v_j / sum w_j / vs,
// so that the weights that meet the codes v_j in 16 bits fit them whatever the scales, the
// largest contribution has full precision, and a block's scale costs one fma that the product s_j
// needs anyway. (Least scale 2^-60: the sum of w / vs stays within 32 bits.)
//
// Rows of a sequence and KV head are (token, query head of the group), G = Hq / Hkv to a token; a
// unit is ROWS of them that share every byte of K and V.
#include <algorithm>
#include <atomic>
#include <climits>

#include "attn_common.hpp"
#include "block8.hpp"
#include "rope.hpp"

namespace sl8 {
namespace {

constexpr int A8_THREADS = 256, A8_WAVES = 4;
constexpr int A8_TILE = 64;       // keys: what splits and units' first keys are multiples of
constexpr int A8_MIN_TILES = 4;   // least keys of a split: a tile for each wave
constexpr float A8_NONE = -1e30f; // reference of nothing
constexpr float A8_LAG = 15.f;    // log2 of the largest weight (fp16 holds it)
constexpr float A8_HEAD = 8.f;    // log2 of a maximum's weight when it becomes the reference

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

struct AttnArgs {
  Block8Seqs s;
  const uint16_t* q;
  const int8_t *k, *v;
  const float *ks, *vs;
  void* out;
  int Hq, Hkv, G;
  float q_mul;
  int window;  // below 0: none
  bool rotate;
  int slots;      // workgroups to split the keys over, 0: no splits
  int whole;      // contexts of up to so many tiles are not split
  int max_pairs;  // that the workspace has places for
  // splits only: partial sums [grid][ROWS][D], (m, l) [grid][ROWS], what to join of each pair
  float* part;
  float2* ml;
  int4* pairs;  // [2 * pairs]: (first item, splits, items between, KV head), (first row, unit's first, rows)
  int* count;   // pairs
};

// ---------------------------------------------------------------------------
// The work list. Every workgroup makes it for itself from the lengths: what is on the device is not
// known to the host, and a launch to make it costs more than these few hundred cycles (a wave
// counts 64 sequences at once).
//
// Items of a sequence: units x Hkv x splits; unsplit calls have room for a unit more a sequence, so
// that where one's begin follows from the offsets alone (1024 of one token on 500 to 3000 keys: 644 us, 681
// with all lengths counted). A split has at most L tiles, L the least for which
// the items fit the slots that are resident at once, so that a batch of mixed lengths gives every
// slot about the same number of keys. KV heads are next to each other: item % 8 is the XCD, and
// the units that read a head's keys meet in its L2.
// ---------------------------------------------------------------------------
struct SeqWork {
  int row0, n, len;  // first row, rows, context
  int units, tiles;
};

struct Item {
  int b, row0, n, len;
  int unit, kvh, split, splits, units, pair;
  int64_t begin, end;  // rows of all sequences
  bool live;
};

template <int ROWS>
__device__ __forceinline__ SeqWork seq_work(const AttnArgs& p, int b) {
  SeqWork w{0, 0, 0, 0, 1};
  if (b < p.s.B) {
    w.row0 = (int)p.s.row(b);
    w.n = max(0, (int)p.s.row(b + 1) - w.row0);
    w.len = p.s.lens[b];
    int span = min(max(w.len, 0), p.s.maxb * p.s.bs);
    if (p.window >= 0) span = (int)min((int64_t)span, (int64_t)p.window + ROWS / p.G + A8_TILE);
    w.units = (w.n * p.G + ROWS - 1) / ROWS;
    w.tiles = max(1, (span + A8_TILE - 1) / A8_TILE);
  }
  return w;
}

// Splits of a sequence: near tiles / L, rounded up (a unit's keys are cut in that many equal parts,
// so a rounding of the quotient leaves nothing out).
__device__ __forceinline__ int splits_of(const AttnArgs& p, int tiles, float over_l) {
  return tiles <= p.whole ? 1 : max(1, (int)ceilf((float)tiles * over_l));
}

// Inclusive sum over the wave: DPP row shifts, then the rows' last lanes.
__device__ __forceinline__ int wave_scan(int x) {
  auto add = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
    x += __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
  };
  using std::integral_constant;
  const integral_constant<int, 0xF> all;
  add(integral_constant<int, 0x111>{}, all);  // row_shr:1
  add(integral_constant<int, 0x112>{}, all);
  add(integral_constant<int, 0x114>{}, all);
  add(integral_constant<int, 0x118>{}, all);
  add(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});  // row_bcast:15
  add(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});  // row_bcast:31
  return x;
}

template <int ROWS>
__device__ __forceinline__ Item find_item(const AttnArgs& p, int lane, int id) {
  if (!p.slots && !p.s.cu) {  // one row a sequence, whole: nothing to look for
    Item it{};
    it.units = (p.G + ROWS - 1) / ROWS;
    const int r = id / p.Hkv;
    it.kvh = id - r * p.Hkv;
    it.b = it.row0 = r / it.units;
    it.unit = r - it.b * it.units;
    it.live = it.b < p.s.B;
    it.n = it.splits = 1;
    it.len = it.live ? p.s.lens[it.b] : 0;
    it.end = p.s.T;
    return it;
  }
  if (!p.slots) {  // whole: units from row0 G / ROWS + b, at least as many as there are
    Item it{};
    it.begin = p.s.row(0);
    it.end = p.s.row(p.s.B);
    const int r = id / p.Hkv;
    const Seq q = seq_of(p.s, lane, r, [&](int row0, int b) { return row0 * p.G / ROWS + b; });
    it.kvh = id - r * p.Hkv;
    it.b = q.b;
    it.row0 = q.row0;
    it.n = q.n;
    it.len = q.len;
    it.splits = 1;
    it.units = (max(q.n, 0) * p.G + ROWS - 1) / ROWS;
    it.unit = it.units - 1 - q.nth;  // (those that see the most keys first)
    it.live = it.unit >= 0;
    return it;
  }
  const SeqWork mine = seq_work<ROWS>(p, lane);
  auto work = [&](int b0) { return b0 == 0 ? mine : seq_work<ROWS>(p, b0 + lane); };
  int most = 1, whole = 0;
  float all = 0.f;
  for (int b0 = 0; b0 < p.s.B; b0 += 64) {
    const SeqWork w = work(b0);
    most = max(most, w.units ? w.tiles : 1);
    whole += w.units;
    all += (float)w.units * (float)w.tiles;
  }
  most = __builtin_amdgcn_readfirstlane(
      (int)lane_group_reduce<64>((uint32_t)most, [](uint32_t a, uint32_t b) { return a > b ? a : b; }));
  whole = __builtin_amdgcn_readfirstlane(lane_group_sum<64>(whole)) * p.Hkv;  // items that none is split
  all = wave_sum(all) * (float)p.Hkv;
  // the least L with items(L) <= slots, four candidates at once
  int lo = __builtin_amdgcn_readfirstlane(max(A8_MIN_TILES, (int)(all / (float)p.slots * 0.999f))), hi = most;
  if (whole < p.slots) hi = min(hi, __builtin_amdgcn_readfirstlane((int)(all / (float)(p.slots - whole))) + 2);
  while (lo < hi) {
    const int step = (hi - lo + 4) / 5 > 1 ? (hi - lo + 4) / 5 : 1;
    int n[4] = {0, 0, 0, 0};
    float r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) r[k] = 1.f / (float)(lo + k * step);
    for (int b0 = 0; b0 < p.s.B; b0 += 64) {
      const SeqWork w = work(b0);
#pragma unroll
      for (int k = 0; k < 4; ++k) n[k] += w.units * splits_of(p, w.tiles, r[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) n[k] = __builtin_amdgcn_readfirstlane(lane_group_sum<64>(n[k])) * p.Hkv;
    int fit = 4;
#pragma unroll
    for (int k = 3; k >= 0; --k)
      if (n[k] <= p.slots) fit = k;
    if (fit < 4) hi = min(hi, lo + fit * step);
    if (fit) lo = min(hi, lo + (fit < 4 ? fit - 1 : 3) * step + 1);
  }
  const float over_l = 1.f / (float)max(lo, 1);
  Item it{};
  int items = 0, pairs = 0;
  for (int b0 = 0; b0 < p.s.B; b0 += 64) {
    const SeqWork w = work(b0);
    const int s = splits_of(p, w.tiles, over_l);
    const int np = w.units * p.Hkv, ni = np * s;
    const int ii = wave_scan(ni), pp = wave_scan(np);
    const uint64_t past = __builtin_amdgcn_ballot_w64(items + ii > id);
    if (past && !it.live) {
      const int at = __builtin_ctzll(past);
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
      it.live = true;
      it.b = b0 + at;
      it.row0 = of(w.row0);
      it.n = of(w.n);
      it.len = of(w.len);
      it.splits = of(s);
      it.units = of(w.units);
      const int r = id - (items + of(ii - ni));
      it.kvh = r % p.Hkv;
      it.unit = it.units - 1 - r / p.Hkv % it.units;  // (those that see the most keys first)
      it.split = r / p.Hkv / it.units;
      it.pair = pairs + of(pp - np) + it.unit * p.Hkv + it.kvh;
      if (id && p.s.B > 64) break;  // (the first workgroup counts all pairs)
    }
    items += __builtin_amdgcn_readlane(ii, 63);
    pairs += __builtin_amdgcn_readlane(pp, 63);
  }
  // (more pairs than places: the offsets fall somewhere, against the contract)
  if (id == 0 && threadIdx.x == 0) *p.count = pairs <= p.max_pairs ? pairs : 0;
  it.begin = __builtin_amdgcn_readlane(mine.row0, 0);
  it.end = p.s.T;
  if (p.s.cu) it.end = p.s.B >= 1 && p.s.B <= 64 ? __builtin_amdgcn_readlane(mine.row0 + mine.n, p.s.B - 1) : p.s.row(p.s.B);
  return it;
}

// The rows and keys of an item.
struct Span {
  int64_t row0;  // first row (token) of the sequence
  int r0, cnt;   // the unit's first of its rows, and how many
  int tok, head; // r0 / G, r0 % G
  float over_g;  // 1 / G
  int pos0;      // position of the sequence's first new token
  int k0, k1;    // keys of the item: from a multiple of a tile
  int low;       // the first key that any row sees
};

// Token (of the sequence's new ones) of a unit's row: (r0 + r) / G. A quotient of less than 2^17 by
// less than 2^16, kept half a row from the next whole number, survives the product's rounding.
__device__ __forceinline__ int token_of(const Span& w, int r) {
  return w.tok + (int)(((float)(w.head + r) + 0.5f) * w.over_g);
}

template <int ROWS>
__device__ __forceinline__ Span item_span(const AttnArgs& p, const Item& it) {
  Span w;
  w.row0 = it.row0;
  const int n = it.n;
  const int64_t len = it.len;
  w.r0 = it.unit * ROWS;
  w.cnt = min(ROWS, n * p.G - w.r0);
  w.tok = w.r0 / p.G;
  w.head = w.r0 - w.tok * p.G;
  w.over_g = 1.f / (float)p.G;
  // (contexts below the new tokens: positions below 0, which see nothing)
  const int64_t pos0 = max(len - n, (int64_t)-(1 << 28));
  w.pos0 = (int)min(pos0, (int64_t)INT_MAX - (1 << 29));
  const int keys = (int)max((int64_t)0, min(len, (int64_t)p.s.maxb * p.s.bs));
  const int last = min(keys, w.pos0 + token_of(w, w.cnt - 1) + 1);
  w.low = p.window >= 0 ? (int)max((int64_t)0, (int64_t)w.pos0 + w.tok - p.window + 1) : 0;
  const int first = w.low & ~(A8_TILE - 1);
  const int tiles = max(0, last - first + A8_TILE - 1) / A8_TILE;
  const int per = (tiles + it.splits - 1) / it.splits * A8_TILE;
  w.k0 = first + it.split * per;
  w.k1 = min(last, w.k0 + per);
  return w;
}

// What the joining kernel needs of a pair (unit, KV head); from its first item.
__device__ __forceinline__ void note_pair(const AttnArgs& p, const Span& w, const Item& it) {
  if (it.pair >= p.max_pairs) return;
  p.pairs[2 * it.pair] = make_int4(blockIdx.x, it.splits, it.units * p.Hkv, it.kvh);
  p.pairs[2 * it.pair + 1] = make_int4((int)w.row0, w.r0, w.cnt, 0);
}

// Rows in front of the first sequence and behind the last are zeros.
__device__ __forceinline__ void zero_rest(const AttnArgs& p, const Item& it, int D) {
  const int64_t n = it.begin + p.s.T - it.end;
  if (n == 0) return;
  const int64_t chunks = (int64_t)p.Hq * D / 8;
  uint4* o = static_cast<uint4*>(p.out);
  for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
    const int64_t t = i < it.begin ? i : it.end + i - it.begin;
    for (int64_t c = threadIdx.x; c < chunks; c += blockDim.x) o[t * chunks + c] = make_uint4(0, 0, 0, 0);
  }
}

// Row r of a unit: its offset in q and out.
__device__ __forceinline__ int64_t row_at(const AttnArgs& p, const Span& w, int kvh, int r, int D) {
  const int t = token_of(w, r);
  return ((w.row0 + t) * p.Hq + kvh * p.G + w.head + r - (t - w.tok) * p.G) * D;
}

// The unit's rows as int8 codes in LDS (row r at place(r)) with their scales (times q_mul); rows past
// the last are zeros.
template <int DT, int D, int ROWS, int THREADS, typename F>
__device__ __forceinline__ void quant_rows(const AttnArgs& p, const Span& w, int kvh, F place, float* qs_s) {
  constexpr int LPR = row_lanes(D), RPB = THREADS / LPR;
  constexpr int N = ROWS / RPB > 4 ? 4 : ROWS / RPB > 1 ? ROWS / RPB : 1;  // rows a thread reads at once
  static_assert(ROWS < RPB || ROWS % (N * RPB) == 0, "whole passes");
  const int lane = threadIdx.x % LPR;
#pragma unroll 1
  for (int r1 = threadIdx.x / LPR; r1 < ROWS; r1 += N * RPB) {
    uint4 raw[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = r1 + i * RPB;
      raw[i] = reinterpret_cast<const uint4*>(p.q + row_at(p, w, kvh, r < w.cnt ? r : 0, D))[lane];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = r1 + i * RPB;
      const bool live = r < w.cnt;
      float f[8];
      VecIO<DT>::unpack(raw[i], f);
      if (p.rotate) hadamard_row<D, DT != SL8_DTYPE_F16>(f, lane);
      float amax = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(f[e]));
      amax = lane_group_max<LPR>(amax);
      const float s = amax * (1.0f / 127.0f), safe = s == 0.f ? 1.f : s;
      const uint2 c = row_codes8<DT>(f, safe);
      reinterpret_cast<uint2*>(place(r))[lane] = live ? c : make_uint2(0, 0);
      if (lane == 0) qs_s[r] = live ? safe * p.q_mul : 0.f;
    }
  }
}

// 16 consecutive keys lie in one block: their first row's offset in the caches and the block's
// scales, none (log2 vs = -inf: weight 0) where there is no block or no key in [low, end).
struct Group {
  int64_t at;  // bytes
  float ks, lv, iv;
};
template <int D>
__device__ __forceinline__ Group key_group(const AttnArgs& p, int b, int kvh, int key, int low, int end) {
  Group g{0, 0.f, -INFINITY, 0.f};
  if (key < end && key + 15 >= low) {
    const int j = key / p.s.bs, off = key - j * p.s.bs;
    const int id = p.s.block(b, j);
    if (id >= 0) {
      const int64_t bh = (int64_t)id * p.Hkv + kvh;
      float vs = p.vs[bh];
      vs = vs < 0x1p-60f ? 0x1p-60f : vs;  // (a block of zeros by any other writer)
      g = Group{(bh * p.s.bs + off) * D, p.ks[bh], __builtin_amdgcn_logf(vs), 1.f / vs};
    }
  }
  return g;
}

__device__ __forceinline__ float lane_value(float x, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

// 8 int8 codes as fp16: byte v xor 0x80 is v + 128, under the exponent byte 0x64 it is 1024 + that.
__device__ __forceinline__ v8h codes_f16(v2i c) {
  h2 o[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = (uint32_t)c[i] ^ 0x80808080u;
    const h2 bias = {(_Float16)1152.f, (_Float16)1152.f};
    o[2 * i] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - bias;
    o[2 * i + 1] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - bias;
  }
  return __builtin_bit_cast(v8h, o);
}

__device__ __forceinline__ float max_xor16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Softmax state of 16 RT rows in the layout of S^T: row 16 rt + col in the lanes of column col.
template <int RT, int D>
struct RowState {
  float qs[RT];
  int lim[RT], low[RT];  // the row sees keys [low, lim)
  int in0, in1;          // keys that every row of the unit sees: [in0, in1)
  float m[RT], l[RT];    // reference (log2) and sum of weights / vs
  v4f o[RT][D / 16];

  __device__ __forceinline__ void init(const AttnArgs& p, const Span& w, int r0, int col, const float* qs_s) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = r0 + 16 * rt + col;
      qs[rt] = qs_s[r];
      const int pos = w.pos0 + token_of(w, min(r, w.cnt - 1));  // (rows past the last: as the last)
      lim[rt] = min(pos + 1, w.k1);
      low[rt] = p.window >= 0 ? (int)max((int64_t)pos - p.window + 1, (int64_t)0) : 0;
      m[rt] = A8_NONE;
      l[rt] = 0.f;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) o[rt][t] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    in1 = min(w.pos0 + w.tok + 1, w.k1);
    in0 = p.window >= 0 ? w.pos0 + token_of(w, w.cnt - 1) - p.window + 1 : 0;
  }

  // Weights of NG groups of 16 keys from their scores (lane (g4, col): keys 16 g + 4 g4 + i from
  // key0): B operands of keys 32 kk + {4 g4 + i, 16 + 4 g4 + i}. The reference m stands 2^A8_HEAD
  // to 2^A8_LAG below the maximum, so that most tiles need no exchange across lanes and no scaling.
  // The largest 16-bit weight is 2^A8_HEAD at least, half a step of the subnormal ones 2^-25: beside its
  // relative 2^-11 a weight is off by 2^-33 of the largest, and one below that is lost. N keys shift
  // the output by N * 2^-33 * 127 vs of the largest contribution at most, whatever that one's own
  // value is (with the maximum as reference, a tail of 2^17 keys of weight 2^-26 behind a value of zero
  // was lost; the two steps of the reference cost 1 %, 3 % in short prompts). The sum takes the weights
  // in 32 bits: in a block of small values a large one may have no 16-bit form beside V's largest.
  // PARTS 2: what the rounding to 16 bits left over, in 16 bits too, as operands of their own.
  template <int NG, int PARTS>
  __device__ __forceinline__ void weights(const v4i (&sc)[RT][NG], const float (&ks)[NG], const float (&lv)[NG],
                                          const float (&iv)[NG], int key0, int keys_end, int g4,
                                          v8h (&wb)[RT][NG / 2][PARTS]) {
    float x[RT][NG][4];
    bool move = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float ref = m[rt] == A8_NONE ? 0.f : m[rt];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float a = qs[rt] * ks[g], c = lv[g] - ref;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[rt][g][i] = fmaf((float)sc[rt][g][i], a, c);
      }
    }
    if (!(key0 >= in0 && keys_end <= in1)) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = key0 + 16 * g + 4 * g4 + i;
            if (key >= lim[rt] || key < low[rt]) x[rt][g][i] = -INFINITY;
          }
    }
    float top[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      top[rt] = -INFINITY;
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) top[rt] = fmaxf(top[rt], x[rt][g][i]);
      move = move || top[rt] > (m[rt] == A8_NONE ? -INFINITY : A8_LAG);
    }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(move) != 0, 0)) {  // the maxima become the references
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const bool none = m[rt] == A8_NONE;
        const float mt = max_xor32(max_xor16(top[rt]));
        const float by = none ? (mt == -INFINITY ? 0.f : mt - A8_HEAD) : fmaxf(mt - A8_HEAD, 0.f);
        m[rt] = none ? (mt == -INFINITY ? A8_NONE : mt - A8_HEAD) : m[rt] + by;
        const float r = none ? 1.f : __builtin_amdgcn_exp2f(-by);
        l[rt] *= r;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) o[rt][d] *= r;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[rt][g][i] -= by;
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_exp2f(x[rt][g][i]);
        l[rt] = fmaf((w[0] + w[1]) + (w[2] + w[3]), iv[g], l[rt]);
        const h2 r[2] = {__builtin_convertvector((v2f{w[0], w[1]}), h2), __builtin_convertvector((v2f{w[2], w[3]}), h2)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const _Float16 hi = r[i / 2][i & 1];
          wb[rt][g / 2][0][4 * (g & 1) + i] = hi;
          if constexpr (PARTS == 2) wb[rt][g / 2][1][4 * (g & 1) + i] = (_Float16)(w[i] - (float)hi);
        }
      }
  }
};

// ---------------------------------------------------------------------------
// Few rows (a decode step, drafted tokens): each wave streams tiles of its own keys for all ROWS
// rows, the 4 waves' states are joined in LDS. Bound by the bytes of K and V.
//   * S^T = K Q^T on v_mfma_i32_16x16x64_i8, K straight from global memory into the A operand
//     (lane (g4, col): 16 bytes of key col), the next tile's loads going out as soon as the
//     products have read this one's;
//   * lane (g4, col) then holds keys 4 g4 + i of each 16 for row col: the softmax needs two
//     exchanges across the wave for the maximum, the weights are the B operand as they are;
//   * V comes by direct copies into a ring of two tiles in LDS and is read transposed
//     (ds_read_b64_tr_b8: 8 keys of a channel), in the order of keys that the weights have, and
//     turned into fp16: O^T += V^T W on v_mfma_f32_16x16x32_f16. 16-byte chunks of a row are
//     placed by an xor of its key, so that the 16 rows of half a wave lie in different banks;
//   * fp16, up to 16 rows: a weight is two fp16 parts, as one alone adds a quarter to what the output's
//     rounding leaves (2.7e-4 for 2.06e-4 relative: 32 sequences of 512 to 8192 keys, 32 / 8 heads). It
//     costs 0.4 of 44.9 us there, 1 of 24.7 at D = 64, 1.7 of 31 for 128 sequences on 1000 keys. One part
//     where it would cost more: 32 rows, whose registers spill already (5 tokens of 16 such
//     sequences 37.6 for 33.4 us), and tiles of many rows, which VALU and MFMA bound; bf16's own
//     rounding hides it (1.70e-3 for 1.68e-3).
// 16 sequences of 32768 tokens, 32 / 8 heads, D = 128, bf16 (1.07 GB): 183 us and 5 for the join, 5.8
// TB/s, the rate of pure reading. 32 of 513 to 8192 tokens (186 MB): 36 and 5; the call takes 44.8 us,
// and 18.6 where each wave stops after its first tile: launches, the work list, the first loads and the
// joins. One of 777: 12.4, all of that kind: the first keys wait for the block's id and scale, and Q,
// whose loads are issued behind theirs, for the keys (the first kernel, a wave for each row and head
// with the codes multiplied one by one, took 20 ms, 5 ms and 258 us).
// ---------------------------------------------------------------------------
template <int D> constexpr int stream_keys() { return D == 256 ? 32 : 64; }
template <int D> __device__ __forceinline__ int v_swizzle(int key) {
  if constexpr (D == 64) return ((key >> 2) & 1) | ((key >> 4) & 1) << 1;
  else if constexpr (D == 128) return ((key >> 1) & 3) | ((key >> 4) & 1) << 2;
  else return (key & 7) | ((key >> 4) & 1) << 3;
}

template <int DT, int D, int RT>
__global__ void __launch_bounds__(A8_THREADS, 2) attn_block8_stream_kernel(const AttnArgs p) {
  constexpr int ROWS = 16 * RT, KT = stream_keys<D>(), NG = KT / 16, KS = D / 64, DTL = D / 16;
  constexpr int TPM = 64 / NG;  // tiles whose groups the lanes hold
  constexpr int PARTS = DT == SL8_DTYPE_F16 && RT == 1 ? 2 : 1;  // of a weight
  // Two arrays, not one of two stages: the compiler sees that the reads of one tile are not of the
  // copies in flight, and waits for none of those. The waves' sums are joined in them (o_place).
  __shared__ __attribute__((aligned(16))) int8_t v0_s[A8_WAVES * KT * D], v1_s[A8_WAVES * KT * D];
  __shared__ __attribute__((aligned(16))) int8_t q_s[ROWS * D];
  __shared__ float qs_s[ROWS], m_s[A8_WAVES][ROWS], l_s[A8_WAVES][ROWS];
  static_assert(ROWS * D * 4 * A8_WAVES <= 2 * A8_WAVES * KT * D, "the sums fit the ring");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g4 = lane >> 4;

  const Item it = find_item<ROWS>(p, lane, blockIdx.x);
  zero_rest(p, it, D);
  if (!it.live) return;
  const Span w = item_span<ROWS>(p, it);
  // places: K's lane in a group, the copies' lanes (16-byte chunk of the row that goes to the
  // lane's place) for even and odd groups, the transposed reads' rows
  const int k_off = col * D + 16 * g4;
  constexpr int CPR = D / 16, CPG = D / 64;  // chunks a row, copies a group
  int v_off[2][CPG];
#pragma unroll
  for (int c = 0; c < CPG; ++c) {
    const int ci = 64 * c + lane, r = ci / CPR, ch = ci % CPR;
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) v_off[odd][c] = r * D + 16 * (ch ^ v_swizzle<D>(16 * odd + r));
  }
  const int vkey = (col >> 1) < 4 ? 4 * g4 + (col >> 1) : 12 + 4 * g4 + (col >> 1);
  const int vt_off = vkey * D + 8 * (col & 1), vt_swz = 16 * v_swizzle<D>(vkey);

  const int first = w.k0 + wave * KT, step = A8_WAVES * KT;
  const int ntiles = first < w.k1 ? (w.k1 - first + step - 1) / step : 0;
  // lane i: group i % NG of the wave's tile i / NG (of each TPM)
  auto groups = [&](int tile) {
    return key_group<D>(p, it.b, it.kvh, first + (tile + lane / NG) * step + 16 * (lane % NG), w.low, w.k1);
  };
  Group cur = groups(0), nxt = cur;
  v4i ka[NG][KS];
  auto base = [&](const Group& g, int i) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)g.at, i);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(g.at >> 32), i);
    return (int64_t)(((uint64_t)hi << 32) | lo);
  };
  auto load = [&](const Group& g, int i0, int8_t* ring) {
    int8_t* const to = ring + wave * KT * D;
#pragma unroll
    for (int g1 = 0; g1 < NG; ++g1) {
      const int64_t at = base(g, i0 + g1);
      const int8_t* kp = p.k + at;
#pragma unroll
      for (int s = 0; s < KS; ++s) ka[g1][s] = *reinterpret_cast<const v4i*>(kp + k_off + 64 * s);
    }
#pragma unroll
    for (int g1 = 0; g1 < NG; ++g1) {
      const brsrc_t vr = make_rsrc(p.v + base(g, i0 + g1), 16 * D);
#pragma unroll
      for (int c = 0; c < CPG; ++c) buf16_to_lds(vr, to + g1 * 16 * D + c * 1024, v_off[g1 & 1][c], 0);
    }
  };
  if (ntiles) load(cur, 0, v0_s);

  quant_rows<DT, D, ROWS, A8_THREADS>(p, w, it.kvh, [&](int r) { return q_s + r * D; }, qs_s);
  __syncthreads();

  v4i qb[RT][KS];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qb[rt][s] = *reinterpret_cast<const v4i*>(q_s + (16 * rt + col) * D + 64 * s + 16 * g4);
  RowState<RT, D> st;
  st.init(p, w, 0, col, qs_s);

  auto tile = [&](int j, const int8_t* ring, int8_t* next) __attribute__((always_inline)) {
    const int i0 = j % TPM * NG;  // the tile's groups are in lanes i0 .. i0 + NG - 1 of cur
    const int key0 = first + j * step;
    if (i0 == 0) nxt = groups(j + TPM);
    v4i sc[RT][NG];
#pragma unroll
    for (int g1 = 0; g1 < NG; ++g1)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        v4i acc = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(ka[g1][s], qb[rt][s], acc, 0, 0, 0);
        sc[rt][g1] = acc;
      }
    float gks[NG], glv[NG], giv[NG];
#pragma unroll
    for (int g1 = 0; g1 < NG; ++g1) {
      gks[g1] = lane_value(cur.ks, i0 + g1);
      glv[g1] = lane_value(cur.lv, i0 + g1);
      giv[g1] = lane_value(cur.iv, i0 + g1);
    }
    // (past the last tile: groups without a block, whose copies read the pool's first rows)
    if (i0 + NG == 64) cur = nxt;
    __builtin_amdgcn_sched_barrier(0);  // (K's registers are taken again, not others beside them)
    load(cur, (i0 + NG) & 63, next);

    v8h wb[RT][NG / 2][PARTS];
    st.weights(sc, gks, glv, giv, key0, key0 + KT, g4, wb);

    // V(j): copied before the NG * KS loads and NG * CPG copies of the next tile
    __builtin_amdgcn_s_waitcnt((((NG * (KS + CPG)) & 15) | ((NG * (KS + CPG)) >> 4) << 14) | 0x0F70);
    __builtin_amdgcn_sched_barrier(0);
    const int8_t* vt = ring + wave * KT * D + vt_off;
    // operands 4 at a time, the next 4 being read under the products: more in flight spill, and so do
    // the places of all, kept over the loop (the empty asm makes them the tile's own)
    int swz = vt_swz;
    asm volatile("" : "+v"(swz));
    auto read = [&](int n) __attribute__((always_inline)) {
      return __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)(
          vt + 32 * (n / DTL) * D + ((16 * (n % DTL)) ^ swz)));
    };
    constexpr int N = NG / 2 * DTL;
    v2i c[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[0][i] = read(i);
#pragma unroll
    for (int n0 = 0; n0 < N; n0 += 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n0 + 4 < N) c[(n0 / 4 + 1) & 1][i] = read(n0 + 4 + i);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v8h a = codes_f16(c[n0 / 4 & 1][i]);
        const int kk = (n0 + i) / DTL, d = (n0 + i) % DTL;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int part = 0; part < PARTS; ++part)
            st.o[rt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, wb[rt][kk][part], st.o[rt][d], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  for (int j = 0; j < ntiles;) {
    tile(j++, v0_s, v1_s);
    if (j >= ntiles) break;
    tile(j++, v1_s, v0_s);
  }

  // ---- join the waves ----
  // 4 channels (chunk c) of a wave's row r: placed by an xor of the row, as a column of rows is written
  constexpr int O_WAVE = ROWS * D * 4, O_FIT = A8_WAVES * KT * D / O_WAVE;  // sums in the first array
  auto o_place = [&](int x, int r, int c) {
    int8_t* a = x < O_FIT ? v0_s + x * O_WAVE : v1_s + (x - O_FIT) * O_WAVE;
    return a + (r * (D / 4) + (c ^ (r & 15))) * 16;
  };
  wait_dma();  // (the copies past the last tile land in the ring that is written below)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    st.l[rt] += __shfl_xor(st.l[rt], 16, 64);
    st.l[rt] += __shfl_xor(st.l[rt], 32, 64);
    if (g4 == 0) {
      m_s[wave][16 * rt + col] = st.m[rt];
      l_s[wave][16 * rt + col] = st.l[rt];
    }
  }
  __syncthreads();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = 16 * rt + col;
    float mm = st.m[rt];
#pragma unroll
    for (int x = 0; x < A8_WAVES; ++x) mm = fmaxf(mm, m_s[x][r]);
    const float f = __builtin_amdgcn_exp2f(st.m[rt] - mm);
#pragma unroll
    for (int d = 0; d < DTL; ++d) *reinterpret_cast<v4f*>(o_place(wave, r, 4 * d + g4)) = st.o[rt][d] * f;
  }
  __syncthreads();
  for (int i = tid; i < ROWS * D / 4; i += A8_THREADS) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    if (r >= w.cnt) break;
    v4f a = *reinterpret_cast<const v4f*>(o_place(0, r, d / 4));
    float mm = m_s[0][r], den = 0.f;
#pragma unroll
    for (int x = 1; x < A8_WAVES; ++x) {
      a += *reinterpret_cast<const v4f*>(o_place(x, r, d / 4));
      mm = fmaxf(mm, m_s[x][r]);
    }
#pragma unroll
    for (int x = 0; x < A8_WAVES; ++x) den += l_s[x][r] * __builtin_amdgcn_exp2f(m_s[x][r] - mm);
    if (it.splits == 1) {
      a *= den > 0.f ? 1.f / den : 0.f;
      const int64_t to = row_at(p, w, it.kvh, r, D) + d;
#pragma unroll
      for (int e = 0; e < 4; ++e) st_out<DT>(p.out, to + e, a[e]);
    } else {
      const int64_t row = (int64_t)blockIdx.x * ROWS + r;
      *reinterpret_cast<v4f*>(p.part + row * D + d) = a;
      if (d == 0) p.ml[row] = make_float2(mm, den);
    }
  }
  if (p.slots && it.split == 0 && tid == 0) note_pair(p, w, it);
}

// ---------------------------------------------------------------------------
// Many rows (prompts, drafts of wide groups): the NW waves of a workgroup have 16 RT rows each and
// share every tile of keys through LDS, two tiles deep: K by direct copies, V turned into fp16
// once on its way (10 instructions for 8 codes, which each wave for itself would spend again). The
// products, the layouts and the softmax are the streaming kernel's; V is read transposed with
// ds_read_b64_tr_b16. One barrier a tile; other workgroups of the CU run across it.
//
// 2048 tokens behind 14336, 32 / 8 heads, D = 128, fp16 (515 GFLOP): 450 us, 1.15 PFLOP/s; its
// products at the rates of large int8 and fp16 ones would take 359. VALU is busy in 65 % of the
// cycles (8 instructions a score, 5 of them conversion, fma, maximum, exp2, sum; 1.2 for V's codes)
// and the matrix pipe in 35 %: they hardly overlap, so every cycle is taken. Measured and not taken: 8 waves a workgroup
// (the same), 32 keys a tile (479), 3 waves a SIMD (spills: 605), products of one tile beside the
// softmax of another in one wave (541), s_setprio around either (490, 500), accumulators that start at
// 1.5 * 2^23 instead of the conversion (442, but logits shift by up to 0.75 of a step of the score).
// 5 tokens of 16 sequences of 1.0 to 16.4 thousand, 64 / 8 heads (40 of 64 rows, 191 MB): 48 us and 6
// for the join. Prompts of 651 to 1301 tokens with a window of 1024, D = 64, 16 / 4 heads: a call of 45 us,
// 22 where each workgroup stops after its first tile (launch, search, Q, that tile, output). K
// and V two tiles ahead through registers instead: 61 us for the 59.5 of the drafts on that box, 46.7 for 45.8.
// ---------------------------------------------------------------------------
template <int D> constexpr int tile_keys() { return D == 256 ? 32 : 64; }
template <int D> __device__ __forceinline__ int k_swizzle(int key) {  // 16-byte chunks, 16 keys apart
  if constexpr (D == 64) return (key >> 2) & 3;
  else if constexpr (D == 128) return (key >> 1) & 7;
  else return key & 15;
}
template <int D> __device__ __forceinline__ int v16_swizzle(int key) {  // 32-byte chunks of fp16 rows
  if constexpr (D == 64) return (key >> 1) & 3;
  else return key & 7;
}

template <int DT, int D, int RT, int NW>
__global__ void __launch_bounds__(64 * NW, 2) attn_block8_tile_kernel(const AttnArgs p) {
  constexpr int THREADS = 64 * NW, ROWS = 16 * RT * NW, KT = tile_keys<D>(), NG = KT / 16;
  constexpr int KS = D / 64, DTL = D / 16, CPR = D / 16;
  constexpr int TPM = 64 / NG;
  constexpr int COPIES = KT * D / (16 * THREADS);  // of 16 bytes a thread, for K and for V
  static_assert(COPIES >= 1 && KT * D % (16 * THREADS) == 0, "a tile in whole copies");
  __shared__ __attribute__((aligned(16))) int8_t k0_s[KT * D], k1_s[KT * D];
  __shared__ __attribute__((aligned(16))) uint16_t v0_s[KT * D], v1_s[KT * D];
  __shared__ float qs_s[ROWS];
  static_assert(ROWS <= 4 * KT, "the rows' codes fit where V will be");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g4 = lane >> 4;
  typedef short v4s __attribute__((ext_vector_type(4)));
  typedef short v8s __attribute__((ext_vector_type(8)));

  const Item it = find_item<ROWS>(p, lane, blockIdx.x);
  zero_rest(p, it, D);
  if (!it.live) return;
  const Span w = item_span<ROWS>(p, it);

  // a thread's copies: 16-byte chunk `ch` of key `key` of the tile (64 threads: one group of 16 keys)
  int k_src[COPIES], v_src[COPIES], v_dst[COPIES];
#pragma unroll
  for (int c = 0; c < COPIES; ++c) {
    const int ci = (c * NW + wave) * 64 + lane, key = ci / CPR, ch = ci % CPR;
    k_src[c] = key % 16 * D + 16 * (ch ^ k_swizzle<D>(key % 16));
    v_src[c] = key % 16 * D + 16 * ch;
    v_dst[c] = key * D + 16 * (ch ^ v16_swizzle<D>(key));
  }
  const int ntiles = w.k0 < w.k1 ? (w.k1 - w.k0 + KT - 1) / KT : 0;
  auto groups = [&](int tile) {
    return key_group<D>(p, it.b, it.kvh, w.k0 + (tile + lane / NG) * KT + 16 * (lane % NG), w.low, w.k1);
  };
  Group cur = groups(0), nxt = cur;
  auto base = [&](int i) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)cur.at, i);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(cur.at >> 32), i);
    return (int64_t)(((uint64_t)hi << 32) | lo);
  };
  uint4 vraw[COPIES];
  auto load = [&](int i0, int8_t* kto) {
#pragma unroll
    for (int c = 0; c < COPIES; ++c) {
      const int64_t at = base(i0 + (c * NW + wave) * 64 / CPR / 16);
      vraw[c] = *reinterpret_cast<const uint4*>(p.v + at + v_src[c]);
      buf16_to_lds(make_rsrc(p.k + at, 16 * D), kto + (c * NW + wave) * 1024, k_src[c], 0);
    }
  };
  auto store_v = [&](uint16_t* vto) {
#pragma unroll
    for (int c = 0; c < COPIES; ++c) {
      const v8h a = codes_f16(v2i{(int)vraw[c].x, (int)vraw[c].y}), b = codes_f16(v2i{(int)vraw[c].z, (int)vraw[c].w});
      *reinterpret_cast<v8h*>(vto + v_dst[c]) = a;
      *reinterpret_cast<v8h*>(vto + v_dst[c] + 8) = b;
    }
  };
  if (ntiles) load(0, k0_s);

  constexpr int FIT = 2 * KT;  // rows of codes in the first array of V
  auto q_place = [&](int r) {
    return r < FIT ? reinterpret_cast<int8_t*>(v0_s) + r * D : reinterpret_cast<int8_t*>(v1_s) + (r - FIT) * D;
  };
  quant_rows<DT, D, ROWS, THREADS>(p, w, it.kvh, q_place, qs_s);
  __syncthreads();
  v4i qb[RT][KS];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qb[rt][s] = *reinterpret_cast<const v4i*>(q_place(16 * (RT * wave + rt) + col) + 64 * s + 16 * g4);
  RowState<RT, D> st;
  st.init(p, w, 16 * RT * wave, col, qs_s);
  __syncthreads();
  if (ntiles) store_v(v0_s);
  wait_dma();
  __syncthreads();

  const int k_swz = k_swizzle<D>(col);
  const int vkey = 4 * g4 + (col >> 2);
  const int vt_off = vkey * D + 4 * (col & 3);                           // (fp16 elements)
  const int vt_swz = 16 * v16_swizzle<D>(vkey);

  auto tile = [&](auto rows, int j, const int8_t* kt, const uint16_t* vt, int8_t* knext, uint16_t* vnext)
      __attribute__((always_inline)) {
    const int i0 = j % TPM * NG;
    const int key0 = w.k0 + j * KT;
    if (i0 == 0) nxt = groups(j + TPM);
    float gks[NG], glv[NG], giv[NG];
#pragma unroll
    for (int g1 = 0; g1 < NG; ++g1) {
      gks[g1] = lane_value(cur.ks, i0 + g1);
      glv[g1] = lane_value(cur.lv, i0 + g1);
      giv[g1] = lane_value(cur.iv, i0 + g1);
    }
    if (i0 + NG == 64) cur = nxt;
    load((i0 + NG) & 63, knext);  // (past the last tile: the pool's first rows)

    if (rows) {
      v4i sc[RT][NG];
#pragma unroll
      for (int g1 = 0; g1 < NG; ++g1) {
        v4i ka[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s)
          ka[s] = *reinterpret_cast<const v4i*>(kt + (16 * g1 + col) * D + 16 * ((4 * s + g4) ^ k_swz));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          v4i acc = {0, 0, 0, 0};
#pragma unroll
          for (int s = 0; s < KS; ++s) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(ka[s], qb[rt][s], acc, 0, 0, 0);
          sc[rt][g1] = acc;
        }
      }
      v8h wb[RT][NG / 2][1];
      st.weights(sc, gks, glv, giv, key0, key0 + KT, g4, wb);

      int swz = vt_swz;
      if (D > 128) asm volatile("" : "+v"(swz));  // (the tile's own: 16 places kept over the loop spill)
#pragma unroll
      for (int kk = 0; kk < NG / 2; ++kk)
#pragma unroll
        for (int d = 0; d < DTL; ++d) {
          const uint16_t* a0 = vt + vt_off + 32 * kk * D + ((16 * d) ^ swz);
          const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(a0));
          const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(a0 + 16 * D));
          const v8h a = __builtin_bit_cast(v8h, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            st.o[rt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, wb[rt][kk][0], st.o[rt][d], 0, 0, 0);
        }
      __builtin_amdgcn_iglp_opt(0);  // reads and products interleaved: 2 % of a long chunk
    }
    store_v(vnext);
    wait_dma();
    __syncthreads();
  };
  auto tiles = [&](auto rows) __attribute__((always_inline)) {
    for (int j = 0; j < ntiles;) {
      tile(rows, j++, k0_s, v0_s, k1_s, v1_s);
      if (j >= ntiles) break;
      tile(rows, j++, k1_s, v1_s, k0_s, v0_s);
    }
  };
  // A wave whose rows lie behind the unit's last has copies to make and no products. 64 rows: a branch
  // in the tile, which also keeps the schedule from taking more registers (138 instead of 162 at
  // D = 128; 40 rows a unit, 191 MB: 58 us, 60 with two loops, 62 without either); 128 rows: two
  // loops, as the branch costs a full unit 2.5 %.
  const bool live = 16 * RT * wave < w.cnt;
  if constexpr (RT == 1) tiles(live);
  else if (live) tiles(std::true_type{});
  else tiles(std::false_type{});

#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float l = st.l[rt];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const int r = 16 * (RT * wave + rt) + col;
    if (r >= w.cnt) continue;
    if (it.splits == 1) {
      const float inv = l > 0.f ? 1.f / l : 0.f;
      uint16_t* to = static_cast<uint16_t*>(p.out) + row_at(p, w, it.kvh, r, D) + 4 * g4;
#pragma unroll
      for (int d = 0; d < DTL; ++d) {
        const v4f a = st.o[rt][d] * inv;
        *reinterpret_cast<uint2*>(to + 16 * d) = make_uint2(pack2<DT>(a[0], a[1]), pack2<DT>(a[2], a[3]));
      }
    } else {
      const int64_t row = (int64_t)blockIdx.x * ROWS + r;
#pragma unroll
      for (int d = 0; d < DTL; ++d) *reinterpret_cast<v4f*>(p.part + row * D + 16 * d + 4 * g4) = st.o[rt][d];
      if (g4 == 0) p.ml[row] = make_float2(st.m[rt], l);
    }
  }
  if (p.slots && it.split == 0 && tid == 0) note_pair(p, w, it);
}

// ---------------------------------------------------------------------------
// The splits of a pair (unit, KV head) joined: a wave per row, D / 64 channels a lane; sums in
// the order of the splits. Bound by the chain of loads: the first partial sums are read beside the
// maxima that weigh them.
// ---------------------------------------------------------------------------
constexpr int JOIN_ROWS = 4, JOIN_4 = 8;
template <int DT, int D, int ROWS>
__global__ void __launch_bounds__(64 * JOIN_ROWS) attn_block8_join_kernel(const AttnArgs p) {
  constexpr int C = D / 64;
  typedef float vc __attribute__((ext_vector_type(C)));
  const int lane = threadIdx.x & 63, r = blockIdx.y * JOIN_ROWS + (threadIdx.x >> 6);
  const int4 a = p.pairs[2 * blockIdx.x], u = p.pairs[2 * blockIdx.x + 1];
  if ((int)blockIdx.x >= *p.count || a.y == 1 || r >= u.z) return;
  const int64_t row0 = (int64_t)a.x * ROWS + r, step = (int64_t)a.z * ROWS;
  auto part = [&](int s) {
    if constexpr (C == 1) return vc{p.part[(row0 + s * step) * D + lane]};
    else return *reinterpret_cast<const vc*>(p.part + (row0 + s * step) * D + C * lane);
  };
  vc x[JOIN_4];
#pragma unroll
  for (int s = 0; s < JOIN_4; ++s) x[s] = part(min(s, a.y - 1));
  float mm = A8_NONE;
  for (int s = lane; s < a.y; s += 64) mm = fmaxf(mm, p.ml[row0 + s * step].x);
  mm = wave_max(mm);
  float den = 0.f;
  vc o = {};
  for (int s0 = 0; s0 < a.y; s0 += 64) {
    float f = 0.f, l = 0.f;
    if (s0 + lane < a.y) {
      const float2 y = p.ml[row0 + (s0 + lane) * step];
      f = __builtin_amdgcn_exp2f(y.x - mm);
      l = y.y * f;
    }
    den += wave_sum(l);
    const int n = min(64, a.y - s0);
    for (int s = 0; s < n; s += JOIN_4) {
      vc y[JOIN_4];
#pragma unroll
      for (int k = 0; k < JOIN_4; ++k)
        if (s0 + s + JOIN_4 < a.y) y[k] = part(min(s0 + s + JOIN_4 + k, a.y - 1));
#pragma unroll
      for (int k = 0; k < JOIN_4; ++k)
        if (s + k < n) o += x[k] * lane_value(f, s + k);
#pragma unroll
      for (int k = 0; k < JOIN_4; ++k) x[k] = y[k];
    }
  }
  const float inv = den > 0.f ? 1.f / den : 0.f;
  const int i = u.y + r;
  const int64_t to = (((int64_t)u.x + i / p.G) * p.Hq + a.w * p.G + i % p.G) * D + C * lane;
#pragma unroll
  for (int c = 0; c < C; ++c) st_out<DT>(p.out, to + c, o[c] * inv);
}

// The kernels by head dim and rows: NW 0 streams.
template <int D_, int RT_, int NW_> struct Shape {
  static constexpr int D = D_, RT = RT_, NW = NW_, ROWS = 16 * RT_ * (NW_ ? NW_ : 1);
  static constexpr int THREADS = NW_ ? 64 * NW_ : A8_THREADS;
  template <int DT> static auto kernel() {
    if constexpr (NW_) return attn_block8_tile_kernel<DT, D, RT, NW>;
    else return attn_block8_stream_kernel<DT, D, RT>;
  }
  // workgroups resident on one CU (asked once)
  static int wgs_per_cu() {
    static std::atomic<int> n{0};
    int v = n.load(std::memory_order_relaxed);
    if (v == 0) {
      if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&v, reinterpret_cast<const void*>(kernel<0>()), THREADS, 0) !=
              hipSuccess || v < 1) {
        (void)hipGetLastError();
        return 2;  // no device: any figure (nothing is launched)
      }
      n.store(v, std::memory_order_relaxed);
    }
    return v;
  }
};

// f(Shape) for `rows` rows of a sequence and KV head on average: what holds them in the fewest units
// without many empty rows, up to 128. Up to 32 rows the waves stream keys of their own. 5 tokens (20 rows)
// of 16 sequences, 32 / 8 heads, D = 128: 33.4 us, 41.6 in tiles of 64 rows, where their lengths go from 517 to
// 8192; 76 and 67 where all have 8192. 64 sequences of 130 to 2000: 38 and 49, all of 2000: 89 and 66. D = 64:
// 21.8 and 36.9, 31.9 and 38.1; 23 and 33, 36 and 42. (The lengths are on the device: mixed ones decide.) 40
// rows (the drafts above) take 57 in tiles, 88 streamed as two units. 32 streamed rows at D = 128 need more
// than the 256 registers of two waves a SIMD: 27 spill (96 to 112 bytes a lane) and come back in the loop
// over keys; 16 rows at D = 256 spill 2, and 32 rows there, whose sums take 128, are not built.
template <typename F>
auto with_shape(int64_t D, int64_t rows, F&& f) {
  auto by_rows = [&](auto d) {
    constexpr int DD = decltype(d)::value;
    if (rows <= 16) return f(Shape<DD, 1, 0>{});
    if constexpr (DD < 256) {
      if (rows <= 32) return f(Shape<DD, 2, 0>{});
    }
    if (rows <= 64) return f(Shape<DD, 1, 4>{});
    return f(Shape<DD, 2, 4>{});
  };
  if (D == 64) return by_rows(std::integral_constant<int, 64>{});
  if (D == 128) return by_rows(std::integral_constant<int, 128>{});
  return by_rows(std::integral_constant<int, 256>{});
}

// How a call runs: a bound on the pairs (unit, KV head), whether keys are split over workgroups, and
// the bytes that that takes.
struct AttnPlan {
  int64_t rows;  // of a sequence and KV head on average
  int64_t pairs;
  int slots, whole;
  int64_t grid;
  size_t bytes;
};

AttnPlan attn_plan(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t keys) {
  AttnPlan a{};
  if (T == 0 || B == 0 || Hq == 0) return a;
  const int64_t G = Hq / Hkv;
  a.rows = (T * G + B - 1) / B;
  with_shape(D, a.rows, [&](auto sh) {
    constexpr int ROWS = decltype(sh)::ROWS;
    a.pairs = Hkv * (T * G / ROWS + B);
    // Splits pay where workgroups would idle, or wait for the longest sequence of a batch, and all
    // pairs fit the slots. With many rows, whose joining costs, only where half the slots may lie idle:
    // full units or sequences for no more than that (8 x 120 tokens on 5000 keys, 32/8 heads: 106 us, 149
    // whole; 512 tokens beside 31 of one on 2 to 6 thousand keys: 79, 115 whole; but 720 pairs of 128
    // rows on 768 slots, D = 64: 48 us whole, 70 split).
    const int64_t slots = (int64_t)cu_count() * decltype(sh)::wgs_per_cu();
    const int64_t least = Hkv * std::max(B, T * G / ROWS);
    // Short contexts stay whole: joining costs a launch (one token on 777 keys, 32/8 heads: 11.9 us whole;
    // 14.7 in a table for 32768, whose call has the work list and the launch), and with many rows 2 D sums
    // of 32 bits for each of them, against a time that goes by D: 300 tokens on 1000 keys (72 of 512
    // slots) 31 us whole, 33 split, on 2000 48 and 38; 4 x 250 (248 slots) on 1200 keys 47 and 53, on 2000
    // 69 and 62; D = 64, 4 x 300 on 2000 37 and 41, on 3000 50 and 47; D = 256, 2 x 180 on 751 52 and 40.
    a.whole = decltype(sh)::NW ? (int)(128 * (12 * slots + 32 * std::min(least, slots)) / (D * slots)) : 16;
    const bool split = keys > a.whole * A8_TILE && a.pairs <= slots && (decltype(sh)::NW == 0 || 2 * least <= slots);
    a.slots = split ? (int)slots : 0;
    a.grid = a.slots ? slots : a.pairs;
    if (a.slots) a.bytes = (size_t)a.grid * ROWS * (D + 2) * 4 + (size_t)a.pairs * 32 + 16;
  });
  return a;
}

}  // namespace
}  // namespace sl8

using namespace sl8;

extern "C" size_t sl8_attn_paged_block8_workspace(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                                                    int64_t max_context_len) {
  // (sizes that the call refuses: nothing to compute, and no quotient by a head dim of 0)
  if (T <= 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || T >= (1LL << 28) || B >= (1 << 24) || Hq >= (1 << 16)) return 0;
  if ((D != 64 && D != 128 && D != 256) || Hq % Hkv) return 0;
  return attn_plan(T, B, Hq, Hkv, D, max_context_len).bytes;
}

extern "C" int sl8_attn_paged_block8(const void* q, int dtype, int rotate, float q_scale_mul,
                                     const int8_t* k_cache, const float* k_scale,
                                     const int8_t* v_cache, const float* v_scale,
                                     const int32_t* cu_lens, const int32_t* context_lens,
                                     const int32_t* block_table, void* out, int64_t T, int64_t B,
                                     int64_t Hq, int64_t Hkv, int64_t D, int64_t num_blocks,
                                     int64_t block_size, int64_t max_blocks_per_seq,
                                     int64_t window_left, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  clear_error();
  const char* tag = "attn_paged_block8";
  SL8_CHECK_ARG(dtype == SL8_DTYPE_F16 || dtype == SL8_DTYPE_BF16, "fni8 %s: q must be float16 or bfloat16", tag);
  SL8_CHECK_ARG(T >= 0 && T < (1LL << 28) && B >= 0 && B < (1 << 24) && Hq >= 0 && Hq < (1 << 16) &&
                    num_blocks >= 0 && num_blocks < (1LL << 31) && max_blocks_per_seq >= 0 &&
                    max_blocks_per_seq < (1LL << 31) && block_size >= 0 && block_size < (1 << 16),
                "fni8 %s: shape too large", tag);
  AttnArgs p{};
  p.s = Block8Seqs{cu_lens, context_lens, block_table, T, (int)B, (int)max_blocks_per_seq, (int)num_blocks,
                   (int)block_size};
  if (const int rc = block8_check(tag, p.s, Hkv, D)) return rc;
  SL8_CHECK_ARG(Hq % Hkv == 0, "fni8 %s: H_q must be divisible by H_kv (GQA)", tag);
  SL8_CHECK_ARG(T * Hq < (1LL << 30) && T * (Hq / Hkv) + B < (1LL << 30) / Hkv, "fni8 %s: shape too large", tag);
  if (T == 0 || Hq == 0) return SL8_OK;
  SL8_CHECK_ARG(q && out && (B == 0 || (context_lens && (max_blocks_per_seq == 0 || block_table))) &&
                    (num_blocks == 0 || (k_cache && k_scale && v_cache && v_scale)),
                "fni8 %s: null pointer", tag);
  SL8_CHECK_ARG(aligned(q, 16) && aligned(out, 16) && aligned(k_cache, 16) && aligned(v_cache, 16),
                "fni8 %s: q/k_cache/v_cache must be 16-byte aligned", tag);
  const AttnPlan plan = attn_plan(T, B, Hq, Hkv, D, max_blocks_per_seq * block_size);
  SL8_CHECK_ARG(plan.grid < (1LL << 32) / A8_THREADS, "fni8 %s: shape too large", tag);
  SL8_CHECK_ARG(plan.bytes == 0 || (workspace && workspace_bytes >= plan.bytes && aligned(workspace, 16)),
                "fni8 %s: workspace needs %zu bytes", tag, plan.bytes);
  p.q = static_cast<const uint16_t*>(q);
  p.k = k_cache; p.v = v_cache; p.ks = k_scale; p.vs = v_scale;
  p.out = out;
  p.Hq = (int)Hq; p.Hkv = (int)Hkv; p.G = (int)(Hq / Hkv);
  p.q_mul = q_scale_mul;
  p.rotate = rotate != 0;
  p.window = window_left < 0 ? -1 : (int)(window_left < (1 << 30) ? window_left : (1 << 30));
  p.slots = plan.slots;
  p.whole = plan.whole;
  p.max_pairs = (int)plan.pairs;
  if (num_blocks == 0) p.s.maxb = 0;  // nothing to read: no key is there
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned grid = (unsigned)(plan.grid > 0 ? plan.grid : 1);
  with_shape(D, plan.rows, [&](auto sh) {
    using S = decltype(sh);
    if (plan.slots) {
      p.pairs = static_cast<int4*>(workspace);
      p.count = reinterpret_cast<int*>(p.pairs + 2 * plan.pairs);
      p.part = reinterpret_cast<float*>(p.count + 4);
      p.ml = reinterpret_cast<float2*>(p.part + (size_t)plan.grid * S::ROWS * D);
    }
    auto go = [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      S::template kernel<DT>()<<<grid, S::THREADS, 0, st>>>(p);
      if (plan.slots)
        attn_block8_join_kernel<DT, S::D, S::ROWS>
            <<<dim3((unsigned)plan.pairs, S::ROWS / JOIN_ROWS), 64 * JOIN_ROWS, 0, st>>>(p);
    };
    if (dtype == SL8_DTYPE_F16) go(std::integral_constant<int, SL8_DTYPE_F16>{});
    else go(std::integral_constant<int, SL8_DTYPE_BF16>{});
  });
  SL8_CHECK_LAUNCH(tag);
  return SL8_OK;
}
