// The 8-bit KV cache: what its kernels share.
//
// Layout: K and V pools [num_pages, n_kv_heads, 16, head_dim] of OCP e4m3 bytes and their scales
// [num_pages, n_kv_heads] as floats, one for each page and kv head ("block"). A block is 1 KiB
// (head_dim 64) or 2 KiB of consecutive memory, read by one wave in whole lines.
//
// A scale is a power of two, 2^-15 to 2^7:
//  * a block whose scale grows (a larger token arrives) is rounded again only where e4m3 runs out
//    of exponents: shifting a floating-point value by powers of two keeps its significand;
//  * every value that a block can hold is an fp16 exactly: the smallest step is 2^-9 * 2^-15 =
//    2^-24, fp16's own, and the largest value 448 * 2^7 = 57344. So v_cvt_scalef32_pk_f16_fp8, which
//    takes the scale along, gives the matrix cores the cached values themselves.
#pragma once

#include "common.hpp"

namespace llmk {
namespace kv8 {

constexpr int kPage = 16;
constexpr float kMaxE4m3 = 448.0f;
constexpr int kMinExp = -15, kMaxExp = 7;

typedef float f32x2 __attribute__((ext_vector_type(2)));

// The rows of a call: sequence s owns rows starts[s] .. starts[s + 1] - 1 (one row each where
// starts is NULL), its last ones: row i of c stands at position lens[s] - c + i.
struct Batch {
  const int* tables;
  const int* starts;
  const int* lens;
  int n_rows, n_seqs, max_pages;
};

// The sequence that row belongs to, -1 if none; the same in every lane. starts[0 .. n_seqs]
// ascends: each step probes 64 entries, so 4096 sequences take two loads one behind the other,
// where halving would take twelve. Reads stay inside the array whatever it holds.
__device__ __forceinline__ int find_seq(const int* __restrict__ starts, int n_seqs, int row) {
  if (!starts) return row < n_seqs ? row : -1;
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n_seqs + 1;
  while (hi - lo > 64) {
    const int step = (hi - lo + 63) / 64;
    const int at = lo + lane * step;
    const int c = __builtin_popcountll(
        __builtin_amdgcn_ballot_w64(at < hi && starts[at < hi ? at : lo] <= row));
    if (c == 0) return -1;
    lo += (c - 1) * step;
    hi = hi < lo + step ? hi : lo + step;
  }
  const int at = lo + lane;
  const int c = __builtin_popcountll(
      __builtin_amdgcn_ballot_w64(at < hi && starts[at < hi ? at : lo] <= row));
  const int s = lo + c - 1;
  return c == 0 || s >= n_seqs ? -1 : s;
}

// The same for one lane, from a sequence that begins at or before row.
__device__ __forceinline__ int find_seq_from(const int* __restrict__ starts, int n_seqs, int lo,
                                             int row) {
  int hi = n_seqs + 1;  // starts[lo] <= row, starts[hi] > row
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (starts[mid] <= row) lo = mid; else hi = mid;
  }
  return lo >= n_seqs ? -1 : lo;
}

__device__ __forceinline__ float exp2_int(int e) {
  return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}
// The exponent of a block's scale, whatever an unwritten one holds.
__device__ __forceinline__ int exponent_of(float scale) {
  const int e = (int)((__builtin_bit_cast(uint32_t, scale) >> 23) & 0xFFu) - 127;
  return e < kMinExp ? kMinExp : e > kMaxExp ? kMaxExp : e;
}

// The least e with most <= 448 * 2^e, within the exponents of a scale: 448 is 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(float most) {
  const uint32_t b = __builtin_bit_cast(uint32_t, most);
  int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  e = e < kMinExp ? kMinExp : e;
  return e > kMaxExp ? kMaxExp : e;
}

// Four values of a block, x = value / scale, as e4m3: to nearest, ties to even; what lies past 448
// (only where the scale's exponent is the largest) is held as 448, NaN and infinities as NaN.
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d) {
  auto in_range = [](float x) {
    const float y = __builtin_fminf(__builtin_fmaxf(x, -kMaxE4m3), kMaxE4m3);
    return __builtin_fabsf(x) < INFINITY ? y : __builtin_nanf("");
  };
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(in_range(a), in_range(b), 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(in_range(c), in_range(d), r, true);
  return (uint32_t)r;
}

// The two values of one half of four e4m3 bytes, as fp16 (exact).
template <bool HIGH>
__device__ __forceinline__ f16x2 from_e4m3(uint32_t bytes, float scale) {
  return __builtin_bit_cast(f16x2,
                            __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, scale, HIGH));
}

}  // namespace kv8
}  // namespace llmk
