// The block-scaled paged int8 cache: codes int8 [num_blocks, Hkv, block_size, D] and one fp32 scale
// per block and head [num_blocks, Hkv], for K and for V; value = code * scale. Sequence b holds
// lens[b] tokens, the j-th in slot j % block_size of block table[b][j / block_size]. New tokens are
// rows of one list: sequence b's are cu[b] .. cu[b + 1] - 1 and the last of its lens[b] (cu absent:
// row b). What these device arrays hold is not known on the host: every use is bounded here.
#pragma once

#include "common.hpp"

namespace sl8 {
namespace {

constexpr int BLK8_MAX = 128;  // largest block size; a multiple of 16

struct Block8Seqs {
  const int32_t* cu;     // [B + 1] or null
  const int32_t* lens;   // [B]
  const int32_t* table;  // [B, maxb]
  int64_t T;
  int B, maxb, num_blocks, bs;

  // first row of sequence b (b = B: past the last)
  __device__ __forceinline__ int64_t row(int b) const {
    if (!cu) return b;
    const int64_t c = cu[b];
    return c < 0 ? 0 : c < T ? c : T;
  }
  __device__ __forceinline__ int block(int b, int j) const {  // -1: none that exists
    if (j >= maxb) return -1;
    const int id = table[(int64_t)b * maxb + j];
    return id >= 0 && id < num_blocks ? id : -1;
  }
};

// The sequence of a unit of work, by a wave: sequence b has the units from first(row(b), b), which rises
// with b. A 64th of the sequences at a step, then one of 64, with all that is asked of it.
struct Seq {
  int b, row0, n, len;  // n = 0: none
  int nth;              // of its units
};
template <typename F>
__device__ __forceinline__ Seq seq_of(const Block8Seqs& s, int lane, int unit, F first) {
  if (s.B == 0) return {};
  int lo = 0, span = s.B;
  while (span > 64) {
    const int step = (span + 63) / 64, b = min(lo + lane * step, s.B - 1);
    const uint64_t le = __builtin_amdgcn_ballot_w64(lane * step < span && first((int)s.row(b), b) <= unit);
    const int at = le ? 63 - __builtin_clzll(le) : 0;
    lo += at * step;
    span = min(step, span - at * step);
  }
  const int b = min(lo + lane, s.B - 1);
  const int row0 = (int)s.row(b), row1 = (int)s.row(b + 1), len = s.lens[b], f = first(row0, b);
  const uint64_t le = __builtin_amdgcn_ballot_w64(lane < span && f <= unit);
  if (le == 0) return {};
  const int at = 63 - __builtin_clzll(le);
  auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
  return {lo + at, of(row0), of(row1) - of(row0), of(len), unit - of(f)};
}

inline int block8_check(const char* tag, const Block8Seqs& s, int64_t Hkv, int64_t D) {
  SL8_CHECK_ARG(D == 64 || D == 128 || D == 256, "fni8 %s: head dim must be 64/128/256, got %lld", tag,
                (long long)D);
  SL8_CHECK_ARG(s.bs >= 16 && s.bs <= BLK8_MAX && s.bs % 16 == 0,
                "fni8 %s: block_size must be a multiple of 16, 16..%d, got %d", tag, BLK8_MAX, s.bs);
  SL8_CHECK_ARG(s.B >= 0 && s.T >= 0 && s.maxb >= 0 && s.num_blocks >= 0 && Hkv > 0 && Hkv < (1 << 16),
                "fni8 %s: bad shape", tag);
  SL8_CHECK_ARG(s.cu || s.T == s.B, "fni8 %s: without cu_lens there is one row per sequence", tag);
  SL8_CHECK_ARG(s.T < (1LL << 28) && s.B < (1 << 24) && (int64_t)s.maxb * s.bs < (1LL << 30),
                "fni8 %s: shape too large", tag);
  return SL8_OK;
}

}  // namespace
}  // namespace sl8
