// kvcache.cu -- the paged HiF4 key/value cache: new rows in (searched encode),
// rows back out as values.
//
// Cache: for K and for V codes (pages, kv_heads, page_size, dh/2) bytes and
// meta (pages, kv_heads, page_size, dh/64) words, the packed unit of hif4x.h
// per 64 elements of a head's row, so a head's tokens of one page lie
// together.  New row `token` of a batch goes to the position its sequence's
// length gives it (find_sequence), the page to pages[seq][position / size].
//
// append_kernel: the searched encode of csrc/codec.cu (six scales, exact
// lv2/lv3 tree, the same roundings and summation order, so the same bits),
// laid out for short batches: eight lanes share a 64-group, lane i owns
// sub-block i in registers.  A thread per group would run the ~5000
// instructions of a group one after another, which is the whole latency of a
// decoding step's append; eight lanes cut that chain to the eighth and read
// 16 bytes each of one 128-byte line.  The group error is summed over the
// sub-blocks left to right by every lane (six chains of eight shuffles).
#include "common.cuh"
#include "hif4_bits.cuh"
#include "hif4_enc.cuh"
#include "kvcache.cuh"
#include "sm100.cuh"

namespace hif4x {

// Index of (row `token`, head) in units of head rows of the cache; -1 where it has no place.
__device__ __forceinline__ int64_t cache_row(const CacheArgs &a, int64_t token, int head, int sub, unsigned mask) {
  const int s = find_sequence(a.cu_new, a.B, token, sub, mask);
  if (s >= a.B || token < (int64_t)a.cu_new[s]) return -1;
  const int64_t pos = (int64_t)a.kv_len[s] - ((int64_t)a.cu_new[s + 1] - token);
  if (pos < 0) return -1;
  const int64_t at = pos >> a.page_shift;
  const int64_t page = at < a.most ? (int64_t)a.pages[s * a.ld_pages + at] : -1;
  if (page < 0 || page >= a.num_pages) {
    atomicExch(a.status + 1, HIF4X_BAD_PAGE);
    return -1;
  }
  return (page * a.heads + head) * a.page_size + (pos & (a.page_size - 1));
}

struct AppendArgs {
  CacheArgs c;
  const void *src[2];
  int64_t ld_row[2], ld_head[2];
  int dtype, vec;   // vec: rows take 16-byte loads
};

// Errors of a sub-block's two quads at the 14 units sig 2^(e0 + m) of the six
// candidate scales: index 4 s + m for s <= 1 (m < 4), 8 + m for s = 2, 11 + m
// for s = 3 (csrc/codec.cu search_fast2, the same operations in the same order).
__device__ __forceinline__ void unit_errors(const float (&x)[8], int e0, float (&Q)[2][14]) {
  const float p2 = exp2i(e0);
  const float u[4] = {p2, __fmul_rn(p2, 1.25f), __fmul_rn(p2, 1.5f), __fmul_rn(p2, 1.75f)};
  const float y[4] = {exp2i(-e0), __fdiv_rn(1.0f, u[1]), __fdiv_rn(1.0f, u[2]), __fdiv_rn(1.0f, u[3])};
  auto qsc = [](int m) { return m == 0 ? 4.0f : m == 1 ? 2.0f : m == 2 ? 1.0f : 0.5f; };
  auto nuq = [&](int s, int m) { return -__fmul_rn(u[s], m == 0 ? 0.25f : m == 1 ? 0.5f : m == 2 ? 1.0f : 2.0f); };
  const u64 Y12 = pk2(y[1], y[2]), NU12 = pk2(-u[1], -u[2]);
  const u64 MAG2 = pk2(kMagic, kMagic), NMAG2 = pk2(-kMagic, -kMagic);
  const u64 QSV[7] = {pk2(qsc(0), qsc(0)), pk2(qsc(1), qsc(1)), pk2(qsc(2), qsc(2)), pk2(qsc(0), qsc(1)),
                      pk2(qsc(2), qsc(3)), pk2(qsc(0), qsc(1)), pk2(qsc(2), qsc(3))};
  const u64 NUV[7] = {pk2(nuq(1, 0), nuq(2, 0)), pk2(nuq(1, 1), nuq(2, 1)), pk2(nuq(1, 2), nuq(2, 2)),
                      pk2(nuq(0, 0), nuq(0, 1)), pk2(nuq(0, 2), nuq(0, 3)), pk2(nuq(3, 0), nuq(3, 1)),
                      pk2(nuq(3, 2), nuq(1, 3))};
  const float M7 = kMagic + 7.0f;
#pragma unroll
  for (int qd = 0; qd < 2; qd++) {
    u64 acc[7];
#pragma unroll
    for (int kk = 0; kk < 4; kk++) {
      const float a = x[4 * qd + kk];
      const u64 a2 = pk2(a, a);
      const float q0 = __fmul_rn(a, y[0]);
      const u64 q12a = mul2(a2, Y12);
      const u64 q12 = fma2(fma2(q12a, NU12, a2), Y12, q12a);
      const float q3a = __fmul_rn(a, y[3]);
      const float q3 = __fmaf_rn(__fmaf_rn(-q3a, u[3], a), y[3], q3a);
      float q1, q2;
      upk2(q12, q1, q2);
      const u64 QIN[7] = {q12, q12, q12, pk2(q0, q0), pk2(q0, q0), pk2(q3, q3), pk2(q3, q1)};
#pragma unroll
      for (int pi = 0; pi < 7; pi++) {
        float tl, th;
        upk2(fma2(QIN[pi], QSV[pi], MAG2), tl, th);
        // scales m = 3 never round above 7: (0,3) and (1,3) skip the clamp
        const u64 t2 = pk2(fminf(tl, M7), (pi == 4 || pi == 6) ? th : fminf(th, M7));
        const u64 d = fma2(add2(t2, NMAG2), NUV[pi], a2);
        const u64 e = mul2(d, d);
        acc[pi] = kk ? add2(acc[pi], e) : e;
      }
    }
    upk2(acc[0], Q[qd][4], Q[qd][8]);
    upk2(acc[1], Q[qd][5], Q[qd][9]);
    upk2(acc[2], Q[qd][6], Q[qd][10]);
    upk2(acc[3], Q[qd][0], Q[qd][1]);
    upk2(acc[4], Q[qd][2], Q[qd][3]);
    upk2(acc[5], Q[qd][11], Q[qd][12]);
    upk2(acc[6], Q[qd][13], Q[qd][7]);
  }
}

// |x| / unit * 4 rounded to even, at most 7, with IEEE division
__device__ __forceinline__ float mant4_ref(float a, float unit) {
  return fminf(rintf(__fmul_rn(__fdiv_rn(a, unit), 4.0f)), 7.0f);
}

// The eight lanes of a group choose its scale: sf and, for this lane's
// sub-block, lv (bit 0 lv2, bits 1-2 the quads' lv3).  Candidate scales that
// meet the E6M2 clamps are evaluated with the divisions of the definition.
__device__ __forceinline__ void choose(const float (&a)[8], float amax, int lane, unsigned mask, float &sf,
                                       uint32_t &lv) {
  const int e0 = floor_log2_torch(fmaxf(__fdiv_rn(amax, 7.0f), 1e-38f));
  const bool fast = e0 >= -48 && e0 <= 14;   // the same in all eight lanes
  const float SIG[6] = {1.0f, 1.25f, 1.5f, 1.75f, 1.0f, 1.25f};
  float Q[2][14];
  if (fast) unit_errors(a, e0, Q);
  const int base = lane & 24;
  float best = 0.0f;
  sf = 0.0f;
  lv = 0;
#pragma unroll
  for (int c = 0; c < 6; c++) {
    const int BASE[6] = {0, 4, 8, 11, 1, 5};
    const float cand = clampf(__fmul_rn(exp2i(e0 + (c >= 4 ? 1 : 0)), SIG[c]), kSfMin, kSfMax);
    float e[2][3];   // per quad, at 1, 2 and 4 times the scale
    if (fast) {
#pragma unroll
      for (int qd = 0; qd < 2; qd++)
#pragma unroll
        for (int m = 0; m < 3; m++) e[qd][m] = Q[qd][BASE[c] + m];
    } else {
#pragma unroll
      for (int qd = 0; qd < 2; qd++)
#pragma unroll
        for (int m = 0; m < 3; m++) {
          const float unit = __fmul_rn(cand, m == 0 ? 1.0f : m == 1 ? 2.0f : 4.0f);
          float s = 0.0f;
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const float v = a[4 * qd + k];
            const float d = __fsub_rn(__fmul_rn(__fmul_rn(mant4_ref(v, unit), 0.25f), unit), v);
            s = __fadd_rn(s, __fmul_rn(d, d));
          }
          e[qd][m] = s;
        }
    }
    // lv3: the smaller unit on ties; lv2: 1 unless 2 is strictly better
    const float ea = __fadd_rn(fminf(e[0][0], e[0][1]), fminf(e[1][0], e[1][1]));
    const float eb = __fadd_rn(fminf(e[0][1], e[0][2]), fminf(e[1][1], e[1][2]));
    const bool two = eb < ea;
    const uint32_t bits = two ? 1u | (e[0][1] > e[0][2] ? 2u : 0u) | (e[1][1] > e[1][2] ? 4u : 0u)
                              : (e[0][0] > e[0][1] ? 2u : 0u) | (e[1][0] > e[1][1] ? 4u : 0u);
    const float mine = two ? eb : ea;
    float err = __shfl_sync(mask, mine, base);
#pragma unroll
    for (int i = 1; i < 8; i++) err = __fadd_rn(err, __shfl_sync(mask, mine, base + i));
    if (c == 0 || err < best) {
      best = err;
      sf = cand;
      lv = bits;
    }
  }
  // A NaN compares with nothing.  With clamped scales the definition
  // (csrc/codec.cu search_generic) keeps the smaller unit where its error is
  // "<=", so a quad with a NaN takes the larger one; without, it takes the
  // larger one where the smaller's error is ">", so there it does not.
  if (!fast) {
    if (!(a[0] + a[1] + a[2] + a[3] >= 0.0f)) lv |= 2u;
    if (!(a[4] + a[5] + a[6] + a[7] >= 0.0f)) lv |= 4u;
  }
}

__global__ void __launch_bounds__(128) append_kernel(const AppendArgs p) {
  const CacheArgs &c = p.c;
  const int lane = threadIdx.x & 31, sub = lane & 7;
  const unsigned mask = 0xffu << (lane & 24);
  const int64_t per = (int64_t)c.heads * c.nb;
  int64_t g = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 3;   // (token, head, 64-group)
  if (g >= c.rows * per) return;
  const int which = blockIdx.y;                                        // K or V
  const int64_t token = g / per;
  const int r = (int)(g - token * per), head = r / c.nb, gi = r - head * c.nb;

  const int64_t at = token * p.ld_row[which] + head * p.ld_head[which] + gi * 64 + sub * 8;
  float x[8];
  if (p.dtype == HIF4X_DT_BF16) {
    const uint16_t *s = static_cast<const uint16_t *>(p.src[which]) + at;
    if (p.vec) {
      const uint4 v = __ldg(reinterpret_cast<const uint4 *>(s));
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; k++) {
        x[2 * k] = __uint_as_float(w[k] << 16);
        x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; k++) x[k] = bf16_bits_to_f32(s[k]);
    }
  } else {
    const float *s = static_cast<const float *>(p.src[which]) + at;
    if (p.vec) {
      const float4 v0 = __ldg(reinterpret_cast<const float4 *>(s)), v1 = __ldg(reinterpret_cast<const float4 *>(s) + 1);
      x[0] = v0.x; x[1] = v0.y; x[2] = v0.z; x[3] = v0.w;
      x[4] = v1.x; x[5] = v1.y; x[6] = v1.z; x[7] = v1.w;
    } else {
#pragma unroll
      for (int k = 0; k < 8; k++) x[k] = s[k];
    }
  }
  const int64_t row = cache_row(c, token, head, sub, mask);
  if (row < 0) return;   // all eight lanes of the group

  float a[8], amax = 0.0f;
  uint32_t nib = 0;
#pragma unroll
  for (int k = 0; k < 8; k++) {
    a[k] = fabsf(x[k]);
    amax = fmaxf(amax, a[k]);
    nib |= (x[k] < 0.0f ? 8u : 0u) << (4 * k);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, o));
  float sf;
  uint32_t lv;
  choose(a, amax, lane, mask, sf, lv);

  uint32_t meta = ((lv & 1u) << (8 + sub)) | ((lv >> 1) << (16 + 2 * sub));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) meta |= __shfl_xor_sync(mask, meta, o);
  // m = min(RNE(|x| / unit * 4), 7) as the codec's packed form computes it: the quotient by sf after Markstein
  // (exact for E6M2 significands), rescaled by the lv factors, clamped at 7.25 and rounded by the magic number
  const float ysf = __fdiv_rn(1.0f, sf);
  const u64 YSF2 = pk2(ysf, ysf), NSF2 = pk2(-sf, -sf), MAG2 = pk2(kMagic, kMagic);
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    const float mq = exp2i(2 - (int)((lv & 1u) + ((lv >> (1 + k / 4)) & 1u)));
    const u64 a2 = pk2(a[k], a[k + 1]), q0 = mul2(a2, YSF2);
    float lo, hi;
    upk2(mul2(fma2(fma2(q0, NSF2, a2), YSF2, q0), pk2(mq, mq)), lo, hi);
    upk2(add2(pk2(fminf(lo, 7.25f), fminf(hi, 7.25f)), MAG2), lo, hi);
    nib |= ((__float_as_uint(lo) & 7u) | ((__float_as_uint(hi) & 7u) << 4)) << (4 * k);
  }
  const int64_t unit = row * c.nb + gi;
  reinterpret_cast<uint32_t *>(c.codes[which])[unit * 8 + sub] = nib;
  if (sub == 0) c.meta[which][unit] = e6m2_code(sf) | meta;
}

struct ReadArgs {
  CacheArgs c;
  void *out[2];
  int dtype;
};

// Rows back out: eight lanes have a (token, head), lane i sub-block i of its
// 64-groups of K and V; the place is looked up once for all of them.
__global__ void __launch_bounds__(128) read_kernel(const ReadArgs p) {
  const CacheArgs &c = p.c;
  const int lane = threadIdx.x & 31, sub = lane & 7;
  const int64_t g = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 3;   // (token, head)
  if (g >= c.rows * c.heads) return;
  const int64_t token = g / c.heads;
  const int64_t row = cache_row(c, token, (int)(g - token * c.heads), sub, 0xffu << (lane & 24));
  if (row < 0) return;
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const int which = u & 1, gi = u >> 1;
    if (gi >= c.nb) break;
    const int64_t unit = row * c.nb + gi;
    const uint32_t w = reinterpret_cast<const uint32_t *>(c.codes[which])[unit * 8 + sub];
    const uint32_t m = c.meta[which][unit];
    uint32_t o[4];
    hif4_decode8<0>(w, Hif4Levels(m, sub), hif4_sf2(m), o);
    const int64_t at = (g * c.nb + gi) * 8 + sub;
    if (p.dtype == HIF4X_DT_BF16) {
      static_cast<uint4 *>(p.out[which])[at] = make_uint4(o[0], o[1], o[2], o[3]);
    } else {
      float4 *d = static_cast<float4 *>(p.out[which]) + 2 * at;
      d[0] = make_float4(__uint_as_float(o[0] << 16), __uint_as_float(o[0] & 0xffff0000u),
                         __uint_as_float(o[1] << 16), __uint_as_float(o[1] & 0xffff0000u));
      d[1] = make_float4(__uint_as_float(o[2] << 16), __uint_as_float(o[2] & 0xffff0000u),
                         __uint_as_float(o[3] << 16), __uint_as_float(o[3] & 0xffff0000u));
    }
  }
}

// Checks a cache and batch description; fills the kernels' arguments.
int cache_args(const hif4x_kv_cache *kv, const hif4x_kv_batch *b, int64_t rows, CacheArgs *a) {
  if (!kv || !b || rows < 0) return HIF4X_ERR_ARG;
  if (!kv->k_codes || !kv->k_meta || !kv->v_codes || !kv->v_meta || kv->num_pages < 1 || kv->kv_heads < 1)
    return HIF4X_ERR_ARG;
  if (!b->cu_new || !b->kv_len || !b->pages || b->sequences < 1 || b->max_pages < 1 || b->ld_pages < b->max_pages)
    return HIF4X_ERR_ARG;
  if ((kv->head_dim != 64 && kv->head_dim != 128) || kv->page_size < 16 || kv->page_size > 256 ||
      (kv->page_size & (kv->page_size - 1)) || kv->kv_heads > 65535)
    return HIF4X_ERR_UNSUPPORTED;
  const uintptr_t al = reinterpret_cast<uintptr_t>(kv->k_codes) | reinterpret_cast<uintptr_t>(kv->v_codes) |
                       reinterpret_cast<uintptr_t>(kv->k_meta) | reinterpret_cast<uintptr_t>(kv->v_meta);
  if (al & 15u) return HIF4X_ERR_ARG;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return HIF4X_ERR_LAUNCH;
  a->codes[0] = static_cast<uint8_t *>(kv->k_codes);
  a->codes[1] = static_cast<uint8_t *>(kv->v_codes);
  a->meta[0] = static_cast<uint32_t *>(kv->k_meta);
  a->meta[1] = static_cast<uint32_t *>(kv->v_meta);
  a->num_pages = kv->num_pages;
  a->heads = kv->kv_heads;
  a->page_size = kv->page_size;
  a->page_shift = __builtin_ctz((unsigned)kv->page_size);
  a->nb = kv->head_dim / 64;
  a->cu_new = b->cu_new;
  a->kv_len = b->kv_len;
  a->pages = b->pages;
  a->B = b->sequences;
  a->most = b->max_pages;
  a->ld_pages = b->ld_pages;
  a->rows = rows;
  a->status = tc::status_words(dev);
  return a->status ? HIF4X_OK : HIF4X_ERR_LAUNCH;
}

// Eight lanes for each of `groups` (row, head, ...), in CTAs of 128; K and V as y where `y` is 2.
static int grid_of(int64_t groups, unsigned y, dim3 *grid) {
  const int64_t blocks = (groups * 8 + 127) / 128;
  if (blocks > INT32_MAX) return HIF4X_ERR_UNSUPPORTED;
  *grid = dim3((unsigned)blocks, y);
  return HIF4X_OK;
}

}  // namespace hif4x

using namespace hif4x;

extern "C" int hif4x_kv_append(const hif4x_kv_cache *kv, const hif4x_kv_batch *batch, const void *k, int64_t k_ld_row,
                               int64_t k_ld_head, const void *v, int64_t v_ld_row, int64_t v_ld_head, int dtype,
                               int64_t rows, void *stream) {
  AppendArgs p{};
  int st = cache_args(kv, batch, rows, &p.c);
  if (st != HIF4X_OK) return st;
  if (rows == 0) return HIF4X_OK;
  if (!k || !v || (dtype != HIF4X_DT_BF16 && dtype != HIF4X_DT_F32)) return HIF4X_ERR_ARG;
  p.src[0] = k;
  p.src[1] = v;
  p.ld_row[0] = k_ld_row;
  p.ld_row[1] = v_ld_row;
  p.ld_head[0] = k_ld_head;
  p.ld_head[1] = v_ld_head;
  p.dtype = dtype;
  const int64_t unit = dtype == HIF4X_DT_BF16 ? 8 : 4;   // elements of a 16-byte load
  p.vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0 && k_ld_row % unit == 0 &&
          k_ld_head % unit == 0 && v_ld_row % unit == 0 && v_ld_head % unit == 0;
  dim3 grid;
  st = grid_of(rows * p.c.heads * p.c.nb, 2, &grid);
  if (st != HIF4X_OK) return st;
  append_kernel<<<grid, 128, 0, (cudaStream_t)stream>>>(p);
  HIF4X_CHECK_LAUNCH();
  return HIF4X_OK;
}

extern "C" int hif4x_kv_read(const hif4x_kv_cache *kv, const hif4x_kv_batch *batch, int64_t rows, void *k, void *v,
                             int dtype, void *stream) {
  ReadArgs p{};
  int st = cache_args(kv, batch, rows, &p.c);
  if (st != HIF4X_OK) return st;
  if (rows == 0) return HIF4X_OK;
  if (!k || !v || (dtype != HIF4X_DT_BF16 && dtype != HIF4X_DT_F32)) return HIF4X_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) return HIF4X_ERR_ARG;
  p.out[0] = k;
  p.out[1] = v;
  p.dtype = dtype;
  dim3 grid;
  st = grid_of(rows * p.c.heads, 1, &grid);
  if (st != HIF4X_OK) return st;
  read_kernel<<<grid, 128, 0, (cudaStream_t)stream>>>(p);
  HIF4X_CHECK_LAUNCH();
  return HIF4X_OK;
}
