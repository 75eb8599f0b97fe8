// hif4_bits.cuh -- packed HiF4 -> bf16 in registers, for the kernels that
// multiply by packed values.
//
// An element is +-(m/4) sf 2^(lv2 + lv3) with m in 0..7 and sf = (4 + M)/4
// 2^E: m (4 + M) <= 49 takes six significant bits, so every HiF4 value is a
// bf16 number and a product with it loses nothing before the fp32 sum.
//
// Decode: a word of eight sign-magnitude nibbles becomes eight offset
// nibbles 8 + v (v = +-m; five integer operations for the word), two of which
// are dropped into the mantissas of a bf16 pair 128 + (8 + v), and one
// bf16x2 FMA takes the offset away and applies the scale:
//   (136 + v) S - 136 S = v S,   S = sf/4 2^(lv2 + lv3),
// exact: 136 S has at most seven significant bits, v S at most six.
// About 3.5 instructions per element with the scales, against 5 and more for
// extracting sign and magnitude one by one.
#pragma once
#include "common.cuh"

namespace hif4x {

// a b + c, kept a multiply-add: shifts and additions in its place would run on
// the ALU pipe, which the masks fill
__device__ __forceinline__ uint32_t mad32(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("mad.lo.u32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// nibbles sign << 3 | m -> 8 + m or 8 - m (no carry leaves a nibble)
__device__ __forceinline__ uint32_t hif4_offset(uint32_t w) {
  const uint32_t neg7 = mad32((w >> 3) & 0x11111111u, 7u, 0u);   // 7 in each negative nibble
  return ((w & 0x77777777u) ^ neg7) + (0x88888888u - neg7);
}

__device__ __forceinline__ uint32_t bf16x2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t bf16x2_mul(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
constexpr uint32_t kNeg136 = 0xc308c308u;   // bf16 pair -136

// bf16 bits of sf/4 in both halves: the E6M2 byte (E + 48) << 2 | M is the
// top of a bf16 significand, so its exponent is rebased by one addition
__device__ __forceinline__ uint32_t hif4_sf2(uint32_t meta) { return mad32(meta & 0xffu, 0x00200020u, 0x26802680u); }

// The lv bits of four sub-blocks i0 .. i0 + 3 of a group: bit j of l2, bits 2j
// and 2j + 1 of l3.
struct Hif4Levels {
  uint32_t l2, l3;
  __device__ __forceinline__ Hif4Levels(uint32_t meta, int i0) : l2(meta >> (8 + i0)), l3(meta >> (16 + 2 * i0)) {}
};
// The scales of sub-block i0 + J (8 elements): quad 0 and quad 1, each in both
// halves.  A bit is moved to both exponents' last place by a multiplication
// (which leaves the ALU pipe, the busier one, to the masks).
template <int J>
__device__ __forceinline__ void hif4_scales(const Hif4Levels &l, uint32_t sf2, uint32_t &s0, uint32_t &s1) {
  static_assert(J >= 0 && J < 4, "four sub-blocks");
  const uint32_t b = mad32(l.l2 & (1u << J), 0x00800080u >> J, sf2);
  s0 = mad32(l.l3 & (1u << (2 * J)), 0x00800080u >> (2 * J), b);
  s1 = mad32(l.l3 & (2u << (2 * J)), 0x00800080u >> (2 * J + 1), b);
}

// The same as one pair: quad 0's scale in the low half, quad 1's in the high one.
template <int J>
__device__ __forceinline__ uint32_t hif4_scale_pair(const Hif4Levels &l, uint32_t sf2) {
  const uint32_t b = mad32(l.l2 & (1u << J), 0x00800080u >> J, sf2);
  return mad32(l.l3 & (1u << (2 * J)), 0x80u >> (2 * J), mad32(l.l3 & (2u << (2 * J)), 0x00800000u >> (2 * J + 1), b));
}

// Word of sub-block i0 + J -> four bf16 pairs in element order (0,1) (2,3) (4,5) (6,7).
template <int J>
__device__ __forceinline__ void hif4_decode8(uint32_t w, const Hif4Levels &l, uint32_t sf2, uint32_t *o) {
  uint32_t s0, s1;
  hif4_scales<J>(l, sf2, s0, s1);
  const uint32_t z0 = bf16x2_mul(s0, kNeg136), z1 = bf16x2_mul(s1, kNeg136);
  const uint32_t lo = hif4_offset(w), hi = lo >> 4;
  // element 2p is nibble 2p (byte p of lo), element 2p + 1 the low nibble of byte p of hi
  o[0] = bf16x2_fma((__byte_perm(lo, hi, 0x0400) & 0x000f000fu) | 0x43004300u, s0, z0);
  o[1] = bf16x2_fma((__byte_perm(lo, hi, 0x0501) & 0x000f000fu) | 0x43004300u, s0, z0);
  o[2] = bf16x2_fma((__byte_perm(lo, hi, 0x0602) & 0x000f000fu) | 0x43004300u, s1, z1);
  o[3] = bf16x2_fma((__byte_perm(lo, hi, 0x0703) & 0x000f000fu) | 0x43004300u, s1, z1);
}

// The same in the order (0,2) (4,6) (1,3) (5,7), two operations cheaper: the
// even and the odd nibbles as bytes, a pair and its exponents by one permute.
template <int J>
__device__ __forceinline__ void hif4_decode8_even_odd(uint32_t w, const Hif4Levels &l, uint32_t sf2, uint32_t *o) {
  uint32_t s0, s1;
  hif4_scales<J>(l, sf2, s0, s1);
  const uint32_t z0 = bf16x2_mul(s0, kNeg136), z1 = bf16x2_mul(s1, kNeg136);
  const uint32_t c = hif4_offset(w), even = c & 0x0f0f0f0fu, odd = (c >> 4) & 0x0f0f0f0fu;
  o[0] = bf16x2_fma(__byte_perm(even, 0x43434343u, 0x4140), s0, z0);
  o[1] = bf16x2_fma(__byte_perm(even, 0x43434343u, 0x4342), s1, z1);
  o[2] = bf16x2_fma(__byte_perm(odd, 0x43434343u, 0x4140), s0, z0);
  o[3] = bf16x2_fma(__byte_perm(odd, 0x43434343u, 0x4342), s1, z1);
}

// Eight packed words and their meta word -> 64 values as bf16 pairs in order.
__device__ __forceinline__ void hif4_decode64(const uint32_t (&w)[8], uint32_t meta, uint32_t (&v)[32]) {
  const uint32_t sf2 = hif4_sf2(meta);
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const Hif4Levels l(meta, 4 * h);
    hif4_decode8<0>(w[4 * h], l, sf2, v + 16 * h);
    hif4_decode8<1>(w[4 * h + 1], l, sf2, v + 16 * h + 4);
    hif4_decode8<2>(w[4 * h + 2], l, sf2, v + 16 * h + 8);
    hif4_decode8<3>(w[4 * h + 3], l, sf2, v + 16 * h + 12);
  }
}

// Where new row `token` of a batch belongs: its sequence (cu_new[s] <= token
// < cu_new[s + 1]) and its position kv_len[s] - (cu_new[s + 1] - token).
// Eight lanes of a warp (aligned, `mask` of them) search together, eight
// pivots a step.  seq = B: behind the last sequence.
__device__ __forceinline__ int find_sequence(const int *cu_new, int B, int64_t token, int sub, unsigned mask) {
  int lo = 0, hi = B;   // the answer: how many of cu_new[1..B] are <= token
  while (lo < hi) {
    const int at = min(hi, lo + 1 + (int)(((int64_t)sub * (hi - lo)) >> 3));
    const unsigned le = __ballot_sync(mask, (int64_t)cu_new[at] <= token) & mask;
    const int n = __popc(le);   // cu_new does not fall, so these are the first n pivots
    const int r = hi - lo;
    const int last = n == 0 ? lo : min(hi, lo + 1 + (int)(((int64_t)(n - 1) * r) >> 3));
    const int next = n == 8 ? hi : min(hi, lo + 1 + (int)(((int64_t)n * r) >> 3)) - 1;
    lo = last;
    hi = max(last, next);
  }
  return lo;
}

}  // namespace hif4x
