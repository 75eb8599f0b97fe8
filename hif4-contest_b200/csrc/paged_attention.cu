// paged_attention.cu -- softmax attention of new tokens over the paged HiF4
// cache: o = sum_t softmax_t(scale q.k_t) v_t over the visible keys t.
//
// Query row j of a sequence of length L with n new rows stands at position
// p = L - n + j and sees the keys t <= p with t > p - window or t < sinks.
//
// attend_rows_kernel (few rows per key head: single tokens, drafts) is bound
// by the cache's bytes and by the instructions that turn them into bf16, so
// it reads each packed byte once, straight into the registers of the thread
// that multiplies it, and keeps no tile in shared memory:
//   S^T = K Q^T, O^T = V^T P^T with mma.m16n8k16: 16 keys (then 16 of the
//   head's dims) are the M side and 8 query rows the N side, so a group of
//   up to 8 query heads wastes no half of the instruction.
//   K: the contraction runs over the dims, whose order is free as long as Q
//   has the same one: thread c of a key's four holds dims c dh/4 .. +dh/4,
//   one 16-byte load, and pairs nibbles j and j + 4 of a word (a shift and a
//   mask, and the pair's scales are the two quads' of one sub-block).
//   V: the contraction runs over keys, so a pair is one dim of two keys: two
//   byte permutes make two words of code pairs out of both keys' words.
// The softmax reference of a row moves only when a score passes it by 2^8:
// weights are then at most 256, and any reference gives the same quotient,
// so the common tile needs one vote and no shuffle and no rescaling.
// A warp takes every fourth 16-key tile of its CTA's share; the warps' sums
// meet in shared memory, the shares of one (sequence, key head) in a second
// kernel that adds them in order (the result does not depend on timing).
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "hif4_bits.cuh"
#include "hif4_enc.cuh"
#include "kvcache.cuh"
#include "sm100.cuh"

namespace hif4x {

// The partial sums of the keys' shares: n shares of `all` rows (of one query
// head) each; n == 1: the result goes out directly.
struct Shares {
  int n;
  int64_t all;
  float *part;   // (n, all, dh)
  float2 *ml;    // (n, all): reference, weight
};

struct AttendArgs {
  CacheArgs c;
  const __nv_bfloat16 *q;
  int64_t q_row, q_head;      // strides in elements, multiples of 8
  __nv_bfloat16 *out;
  int64_t o_row, o_head;
  int group;                  // query heads per key head
  float scale;                // times log2(e)
  int window, sinks;          // window 0: all keys
  int most_rows;              // attend_rows_kernel: sequences of up to so many rows; attend_tiles_kernel: of more
  Shares sh;
  int slots;                  // attend_rows_kernel: 0: its sums lie by (token, query head), else by (sequence, key head, row)
  float2 *mark;               // attend_rows_kernel: the other kernel's first pairs, whose weight -1 says that a row is not its
};

// Rows (token, query head of a key head) that the call's tensors have of a
// sequence with n_new rows from cu0 on: the batch may be described beyond them.
__device__ __forceinline__ int64_t rows_present(const AttendArgs &a, int cu0, int n_new) {
  if (n_new <= 0 || cu0 < 0 || cu0 >= a.c.rows) return 0;
  return min((int64_t)n_new, a.c.rows - cu0) * a.group;
}

// Rows of a sequence and key head up to which attend_rows_kernel takes them
// where both kernels run.
constexpr int FEW_ROWS = 16;

constexpr int64_t MOST_SPLITS = 64;   // shares of a row's keys (attend_join_kernel: four warps, a lane for each of 16)
constexpr float kLazy = 8.0f;    // log2 a row's scores may pass its reference by

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// hif4_scales and hif4_scale_pair of sub-block j, an index that unrolling makes constant
__device__ __forceinline__ void scales_of(const Hif4Levels &l, uint32_t sf2, int j, uint32_t &s0, uint32_t &s1) {
  if (j == 0) hif4_scales<0>(l, sf2, s0, s1);
  else if (j == 1) hif4_scales<1>(l, sf2, s0, s1);
  else if (j == 2) hif4_scales<2>(l, sf2, s0, s1);
  else hif4_scales<3>(l, sf2, s0, s1);
}

__device__ __forceinline__ uint32_t scale_pair_of(const Hif4Levels &l, uint32_t sf2, int j) {
  return j == 0 ? hif4_scale_pair<0>(l, sf2) : j == 1 ? hif4_scale_pair<1>(l, sf2)
       : j == 2 ? hif4_scale_pair<2>(l, sf2) : hif4_scale_pair<3>(l, sf2);
}

// The 16-key tiles a run of positions [p_lo, p_hi] of one sequence can see:
// the sinks' tiles, then those from the window's first key to p_hi.
struct KeyTiles {
  int n_sink, n, first;   // tiles; the first window tile
  __device__ __forceinline__ KeyTiles(int p_lo, int p_hi, int window, int sinks, int tile) {
    first = 0;
    n_sink = 0;
    if (p_hi < 0) {
      n = 0;
      return;
    }
    if (window > 0 && p_lo - window + 1 > 0) {
      first = (p_lo - window + 1) / tile;
      n_sink = min(first, (sinks + tile - 1) / tile);
    }
    n = n_sink + p_hi / tile - first + 1;
  }
  __device__ __forceinline__ int key0(int i, int tile) const { return (i < n_sink ? i : i - n_sink + first) * tile; }
};

// One 16-key tile's packed words in registers, and where this lane's lie
// within the 16 rows of a tile.
template <int DH>
struct TileRegs {
  uint32_t k[2][DH / 32], km[2], v[4][DH / 64], vm[4];
  const uint8_t *kc, *vc;
  const uint32_t *kp, *vp;

  __device__ __forceinline__ TileRegs(const CacheArgs &c, int lane) {
    const int n = lane >> 2, q = lane & 3;
    kc = c.codes[0] + n * (DH / 2) + q * (DH / 8);
    kp = c.meta[0] + n * (DH / 64) + (DH == 128 ? q >> 1 : 0);
    vc = c.codes[1] + 2 * q * (DH / 2) + n * (DH / 16);
    vp = c.meta[1] + 2 * q * (DH / 64) + (DH == 128 ? n >> 2 : 0);
  }
  // rows n8 and n8 + 8 of the tile, this thread's quarter of the dims
  __device__ __forceinline__ void load_k(int64_t row) {
    const uint8_t *src = kc + row * (DH / 2);
    const uint32_t *meta = kp + row * (DH / 64);
#pragma unroll
    for (int u = 0; u < 2; u++) {
      if (DH == 128) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4 *>(src + u * 8 * (DH / 2)));
        k[u][0] = w.x;
        k[u][1] = w.y;
        k[u][DH / 32 - 2] = w.z;
        k[u][DH / 32 - 1] = w.w;
      } else {
        const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(src + u * 8 * (DH / 2)));
        k[u][0] = w.x;
        k[u][1] = w.y;
      }
      km[u] = __ldcs(meta + u * 8 * (DH / 64));
    }
  }
  // rows 2 q4, + 1, + 8, + 9, this thread's eighth of the dims
  __device__ __forceinline__ void load_v(int64_t row) {
    const uint8_t *src = vc + row * (DH / 2);
    const uint32_t *meta = vp + row * (DH / 64);
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int r = (u & 1) + 8 * (u >> 1);
      if (DH == 128) {
        const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(src + r * (DH / 2)));
        v[u][0] = w.x;
        v[u][DH / 64 - 1] = w.y;
      } else {
        v[u][0] = __ldcs(reinterpret_cast<const uint32_t *>(src + r * (DH / 2)));
      }
      vm[u] = __ldcs(meta + r * (DH / 64));
    }
  }
};

// DH: head dim; NT: query rows / 8 of a row tile.
template <int DH, int NT>
__global__ void __launch_bounds__(128, NT == 1 ? 3 : 2) attend_rows_kernel(const AttendArgs a) {
  constexpr int WARPS = 4, KW = DH / 32, ROWS = 8 * NT;
  __shared__ float so[WARPS][ROWS][DH + 4];
  __shared__ float2 sml[WARPS][ROWS];
  const CacheArgs &c = a.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n8 = lane >> 2, q4 = lane & 3;
  const int s = blockIdx.x, kh = blockIdx.y, split = blockIdx.z;
  const int cu0 = c.cu_new[s], n_new = c.cu_new[s + 1] - cu0;
  const int64_t rows = rows_present(a, cu0, n_new);
  if (rows == 0 || (int64_t)n_new * a.group > a.most_rows) return;
  const int64_t room = (int64_t)c.most << c.page_shift;
  const int old = c.kv_len[s] - n_new;   // position of the first new row
  const int *pages = c.pages + s * c.ld_pages;

  for (int64_t r0 = 0; r0 < rows; r0 += ROWS) {
    const int64_t r1 = min(rows, r0 + ROWS);
    const int p_lo = old + (int)(r0 / a.group);
    const int p_top = old + (int)((r1 - 1) / a.group);
    int p_hi = p_top;
    if (p_hi >= room) {   // the table has no page for its last keys
      if (threadIdx.x == 0) atomicExch(c.status + 1, HIF4X_BAD_PAGE);
      p_hi = (int)(room - 1);
    }
    // this thread's Q fragments: row r0 + 8 nt + n8, dims q4 dh/4 .. in pairs (j, j + 4)
    uint32_t qf[NT][KW * 4];
    int pos[NT][2];   // positions of the rows 8 nt + 2 q4 + {0, 1} whose scores this thread has
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int64_t r = r0 + 8 * nt + n8;
      const int64_t token = (int64_t)cu0 + r / a.group;
      const bool ok = r < r1 && token >= 0 && token < c.rows;
      const uint4 *src = reinterpret_cast<const uint4 *>(
          a.q + (ok ? token * a.q_row + (kh * a.group + (int)(r % a.group)) * a.q_head + q4 * (DH / 4) : 0));
#pragma unroll
      for (int w = 0; w < KW; w++) {
        const uint4 x = ok ? __ldg(src + w) : make_uint4(0, 0, 0, 0);   // dims 8w .. 8w + 7
        qf[nt][4 * w + 0] = __byte_perm(x.x, x.z, 0x5410);
        qf[nt][4 * w + 1] = __byte_perm(x.x, x.z, 0x7632);
        qf[nt][4 * w + 2] = __byte_perm(x.y, x.w, 0x5410);
        qf[nt][4 * w + 3] = __byte_perm(x.y, x.w, 0x7632);
      }
#pragma unroll
      for (int b = 0; b < 2; b++) {
        const int64_t rr = r0 + 8 * nt + 2 * q4 + b;
        pos[nt][b] = rr < r1 ? old + (int)(rr / a.group) : -1;
      }
    }
    float o[DH / 16][NT][4], ref[NT][2], sum[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int b = 0; b < 2; b++) {
        ref[nt][b] = -INFINITY;
        sum[nt][b] = 0.0f;
      }
#pragma unroll
      for (int mt = 0; mt < DH / 16; mt++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[mt][nt][e] = 0.0f;
    }

    const KeyTiles tiles(min(max(p_lo, 0), p_hi), p_hi, a.window, a.sinks, 16);
    const int per = (tiles.n + a.sh.n - 1) / a.sh.n;
    const int t1 = min(tiles.n, (split + 1) * per);
    int t = split * per + warp;
    // the page of a tile two ahead, the words of the next one
    auto page_of = [&](int i) -> int {
      if (i >= t1) return -1;
      const int pg = __ldg(pages + (tiles.key0(i, 16) >> c.page_shift));
      if (pg >= 0 && pg < c.num_pages) return pg;
      if (lane == 0) atomicExch(c.status + 1, HIF4X_BAD_PAGE);
      return -1;
    };
    auto row_of = [&](int i, int pg) -> int64_t {
      return ((int64_t)pg * c.heads + kh) * c.page_size + (tiles.key0(i, 16) & (c.page_size - 1));
    };
    TileRegs<DH> cur(c, lane);
    int pg = page_of(t), pg_next = page_of(t + WARPS);
    if (pg >= 0) {
      cur.load_k(row_of(t, pg));
      cur.load_v(row_of(t, pg));
    }
    // Two tiles a turn: the words loaded ahead need no moves between registers
    // (64 sequences of up to 8192 keys: 169 us, one a turn 177; three and four
    // a turn 195 and 250).
#pragma unroll 2
    for (; t < t1; t += WARPS) {
      const int pg_next2 = page_of(t + 2 * WARPS);
      const int64_t row_next = pg_next >= 0 ? row_of(t + WARPS, pg_next) : 0;
      if (pg >= 0) {
        const int key0 = tiles.key0(t, 16);
        // ---- scores: S^T (16 keys x 8 NT rows)
        float sc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) sc[nt][e] = 0.0f;
        const uint32_t sf0 = hif4_sf2(cur.km[0]), sf1 = hif4_sf2(cur.km[1]);
        const int i0 = DH == 128 ? (q4 & 1) * 4 : q4 * 2;   // sub-block of the group
        const Hif4Levels l0(cur.km[0], i0), l1(cur.km[1], i0);
#pragma unroll
        for (int w = 0; w < KW; w++) {
          const uint32_t s0 = scale_pair_of(l0, sf0, w), s1 = scale_pair_of(l1, sf1, w);
          const uint32_t z0 = bf16x2_mul(s0, kNeg136), z1 = bf16x2_mul(s1, kNeg136);
          const uint32_t x0 = hif4_offset(cur.k[0][w]), x1 = hif4_offset(cur.k[1][w]);
          uint32_t f[4][2];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            f[j][0] = bf16x2_fma(((x0 >> (4 * j)) & 0x000f000fu) | 0x43004300u, s0, z0);
            f[j][1] = bf16x2_fma(((x1 >> (4 * j)) & 0x000f000fu) | 0x43004300u, s1, z1);
          }
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const uint32_t fa[4] = {f[2 * h][0], f[2 * h][1], f[2 * h + 1][0], f[2 * h + 1][1]};
#pragma unroll
            for (int nt = 0; nt < NT; nt++) mma_bf16(sc[nt], fa, qf[nt][4 * w + 2 * h], qf[nt][4 * w + 2 * h + 1]);
          }
        }
        if (pg_next >= 0) cur.load_k(row_next);   // K's registers are free again; V's after the second product
        // ---- mask; scores to log2 units.  sc[e]: key key0 + n8 + 8 (e >> 1), row 8 nt + 2 q4 + (e & 1)
        const bool all = key0 + 15 <= p_lo && (a.window == 0 || key0 > p_top - a.window || key0 + 15 < a.sinks);
        bool over = false;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            sc[nt][e] *= a.scale;
            if (!all) {
              const int key = key0 + n8 + 8 * (e >> 1), p = pos[nt][e & 1];
              if (!(key <= p && (a.window == 0 || key > p - a.window || key < a.sinks))) sc[nt][e] = -INFINITY;
            }
            over |= sc[nt][e] > ref[nt][e & 1] + kLazy;
          }
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int b = 0; b < 2; b++) {
              float m = fmaxf(ref[nt][b], fmaxf(sc[nt][b], sc[nt][2 + b]));
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
              const float f = ref[nt][b] == -INFINITY ? 0.0f : ex2(ref[nt][b] - m);
              ref[nt][b] = m;
              sum[nt][b] *= f;
#pragma unroll
              for (int mt = 0; mt < DH / 16; mt++) {
                o[mt][nt][b] *= f;
                o[mt][nt][2 + b] *= f;
              }
            }
        }
        // ---- weights, transposed for the second product.  They go to bf16 there, which is off by half a step (2^-8 of
        // a weight at most) from key to key alike: about the size of the result's own rounding (against 64 bits 0.0022
        // of the result where the rounding alone gives 0.0016).  A low part beside it would be a second product over
        // V, whose decoded pairs are in registers for one.  The weights' sum stays fp32.
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float m = ref[nt][e & 1];
            p[e] = ex2(sc[nt][e] - (m == -INFINITY ? 0.0f : m));
            sum[nt][e & 1] += p[e];
          }
          pb[nt][0] = transpose8x8(pack_bf16(p[0], p[1]));
          pb[nt][1] = transpose8x8(pack_bf16(p[2], p[3]));
        }
        // ---- O^T (dh x 8 NT) += V^T P^T
        uint32_t vsf[4];
#pragma unroll
        for (int u = 0; u < 4; u++) vsf[u] = hif4_sf2(cur.vm[u]);
#pragma unroll
        for (int w = 0; w < DH / 64; w++) {
          uint32_t sk[4][2], x[4];
#pragma unroll
          for (int u = 0; u < 4; u++) {
            scales_of(Hif4Levels(cur.vm[u], DH == 128 ? (n8 & 3) * 2 : n8), vsf[u], w, sk[u][0], sk[u][1]);
            x[u] = hif4_offset(cur.v[u][w]);
          }
#pragma unroll
          for (int h = 0; h < 2; h++) {   // quad: dims 4h .. 4h + 3 of the word
            const uint32_t s01 = __byte_perm(sk[0][h], sk[1][h], 0x5410), s23 = __byte_perm(sk[2][h], sk[3][h], 0x5410);
            const uint32_t z01 = bf16x2_mul(s01, kNeg136), z23 = bf16x2_mul(s23, kNeg136);
            const uint32_t y01 = __byte_perm(x[0], x[1], h ? 0x7632 : 0x5410);
            const uint32_t y23 = __byte_perm(x[2], x[3], h ? 0x7632 : 0x5410);
#pragma unroll
            for (int j = 0; j < 2; j++) {
              const uint32_t fa[4] = {
                  bf16x2_fma(((y01 >> (8 * j)) & 0x000f000fu) | 0x43004300u, s01, z01),
                  bf16x2_fma(((y01 >> (8 * j + 4)) & 0x000f000fu) | 0x43004300u, s01, z01),
                  bf16x2_fma(((y23 >> (8 * j)) & 0x000f000fu) | 0x43004300u, s23, z23),
                  bf16x2_fma(((y23 >> (8 * j + 4)) & 0x000f000fu) | 0x43004300u, s23, z23)};
#pragma unroll
              for (int nt = 0; nt < NT; nt++) mma_bf16(o[w * 4 + h * 2 + j][nt], fa, pb[nt][0], pb[nt][1]);
            }
          }
        }
      }
      else if (pg_next >= 0) cur.load_k(row_next);
      if (pg_next >= 0) cur.load_v(row_next);
      pg = pg_next;
      pg_next = pg_next2;
    }

    // ---- the four warps' sums: row 8 nt + 2 q4 + b, dims n8 dh/8 + 2 mt + {0, 1}
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int b = 0; b < 2; b++) {
        float l = sum[nt][b];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
        const int r = 8 * nt + 2 * q4 + b;
        if (n8 == 0) sml[warp][r] = make_float2(ref[nt][b], l);
#pragma unroll
        for (int mt = 0; mt < DH / 16; mt++)
          *reinterpret_cast<float2 *>(&so[warp][r][n8 * (DH / 8) + 2 * mt]) = make_float2(o[mt][nt][b], o[mt][nt][2 + b]);
      }
    __syncthreads();
    for (int e = threadIdx.x; e < ROWS * (DH / 4); e += 128) {
      const int r = e / (DH / 4), d = (e % (DH / 4)) * 4;
      const int64_t rr = r0 + r, token = (int64_t)cu0 + rr / a.group;
      if (rr >= r1 || token < 0 || token >= c.rows) continue;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; w++) m = fmaxf(m, sml[w][r].x);
      float l = 0.0f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WARPS; w++) {
        const float2 ml = sml[w][r];
        const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - m);
        l += f * ml.y;
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] += f * so[w][r][d + k];
      }
      const int head = kh * a.group + (int)(rr % a.group);
      if (a.mark != nullptr && split == 0 && d == 0) a.mark[token * (c.heads * a.group) + head] = make_float2(0.0f, -1.0f);
      if (a.sh.n == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        *reinterpret_cast<uint2 *>(a.out + token * a.o_row + head * a.o_head + d) =
            make_uint2(pack_bf16(v[0] * inv, v[1] * inv), pack_bf16(v[2] * inv, v[3] * inv));
      } else {
        const int64_t at = split * a.sh.all + (a.slots ? ((int64_t)s * c.heads + kh) * FEW_ROWS + rr
                                                       : token * (c.heads * a.group) + head);
        *reinterpret_cast<float4 *>(a.sh.part + at * DH + d) = make_float4(v[0], v[1], v[2], v[3]);
        if (d == 0) a.sh.ml[at] = make_float2(m, l);
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- many rows
// attend_tiles_kernel (prefill chunks) is bound by the tensor cores, the
// exponentials and the instructions around them.  A CTA takes 256 rows
// (token, query head) of one key head as two tiles of 128 and walks the keys
// 128 at a time:
//   warps 0-3, 4-7  softmax of tile 0 and 1: a thread is one row; S from
//                   tensor memory, weights back as bf16 pairs over S, where
//                   the second product reads its A operand
//   warps 8, 9      one lane each issues a tile's products (tcgen05.mma kind::f16):
//                   S = Q K^T (K-major K) and O += P V (V as it lies, keys by
//                   dims: an MN-major B operand, so nothing is transposed)
//   warps 12-19     decode the packed K and V tiles to bf16 in shared memory,
//                   two stages each, the next tile's words in registers
// S0 S1 O0 O1 fill the 512 columns at dh 128 and the weights lie over their
// scores, so the softmax goes by half steps of 64 keys: a tile's two halves
// are two buffers, and while one is in the softmax the tensor core finishes
// the other's second product and computes its next scores.  (With one buffer
// of 128 keys a tile's softmax and products ran one after the other: a
// 2048-token chunk over 10240 keys took 447 us, now 380.)  The softmax
// reference moves as in attend_rows_kernel, only past 2^8; then the row's O
// is rescaled in tensor memory by the softmax warp, once the product before
// has finished.
namespace tiles {

using namespace tc;

constexpr int THREADS = 640, KEYS = 128, ROWS = 256;

template <int DH>
struct Cfg {
  static constexpr int TILE = 128 * DH * 2;                 // bytes of a 128-row bf16 tile
  static constexpr int PANEL = 128 * 128;                   // 64 dims of it
  static constexpr int Q = 0, K = 2 * TILE, V = 4 * TILE;   // two Q tiles, two stages of K and of V
  static constexpr int BARS = 6 * TILE;
  static constexpr int SMEM = BARS + 512 + 1024;
};

// A warp's 16 keys of a K or V tile, packed in registers: lane -> (key of a
// run of eight or sixteen, 16-byte chunk of 32 dims).
template <int DH>
struct Words {
  static constexpr int CPR = DH / 32;          // chunks per row
  static constexpr int KPI = 32 / CPR;         // keys per load
  static constexpr int N = 16 / KPI;           // loads
  uint4 w[N];
  uint32_t m[N];
};

template <int DH>
struct Loader {
  using W = Words<DH>;
  int key, part;                  // key of a load, first sub-block of the lane's half group
  uint32_t codes_at, meta_at;     // bytes from a 16-key block's first row
  uint32_t page_codes, page_meta; // bytes of a page (all heads)
  uint32_t head_codes, head_meta; // bytes to this head's rows in it
  int slots;                      // page_size - 1
  uint32_t to;                    // byte of the lane's first row in a tile

  __device__ __forceinline__ Loader(const CacheArgs &c, int kh, int warp, int lane) {
    const int chunk = W::CPR == 4 ? lane >> 3 : (lane >> 3) & 1;
    key = (lane & 7) + (W::CPR == 2 ? 8 * (lane >> 4) : 0);
    part = (chunk & 1) * 4;
    codes_at = key * (DH / 2) + chunk * 16;
    meta_at = (key * (DH / 64) + (W::CPR == 4 ? chunk >> 1 : 0)) * 4;
    page_codes = (uint32_t)c.heads * c.page_size * (DH / 2);
    page_meta = (uint32_t)c.heads * c.page_size * (DH / 64) * 4;
    head_codes = (uint32_t)kh * c.page_size * (DH / 2);
    head_meta = (uint32_t)kh * c.page_size * (DH / 64) * 4;
    slots = c.page_size - 1;
    to = (W::CPR == 4 ? (chunk >> 1) * Cfg<DH>::PANEL : 0) + (warp * 16 + key) * 128;
  }
  // keys first .. first + 15, all of page `page`.  Where there is none (negative) page 0's are taken, and keys
  // behind the last come as they lie there: every bit pattern decodes to a finite value, and their scores are
  // masked, so nothing of them reaches a result.
  __device__ __forceinline__ void load(W &x, const uint8_t *codes, const uint32_t *meta, int first, int page) const {
    const uint32_t p = (uint32_t)max(page, 0), slot = (uint32_t)(first & slots);
    const uint8_t *src = codes + (uint64_t)p * page_codes + (head_codes + slot * (DH / 2) + codes_at);
    const uint8_t *msrc = reinterpret_cast<const uint8_t *>(meta) + (uint64_t)p * page_meta + (head_meta + slot * (DH / 16) + meta_at);
#pragma unroll
    for (int it = 0; it < W::N; it++) {
      x.w[it] = __ldg(reinterpret_cast<const uint4 *>(src + it * W::KPI * (DH / 2)));
      x.m[it] = __ldg(reinterpret_cast<const uint32_t *>(msrc + it * W::KPI * (DH / 16)));
    }
  }
  // decoded into a tile: panel of 64 dims, key rows of 128 bytes, 16-byte chunk q at q ^ (key & 7); inside a
  // chunk the dims stand as (0 2 4 6 1 3 5 7), as Q's do
  __device__ __forceinline__ void store(const W &x, uint8_t *tile) const {
    uint8_t *row = tile + to;
    const int swz = key & 7;
#pragma unroll
    for (int it = 0; it < W::N; it++) {
      const uint32_t sf2 = hif4_sf2(x.m[it]);
      const Hif4Levels l(x.m[it], part);
      const uint4 c = x.w[it];
      uint8_t *at = row + it * W::KPI * 128;
      uint32_t o[4];
      hif4_decode8_even_odd<0>(c.x, l, sf2, o);
      *reinterpret_cast<uint4 *>(at + ((part ^ swz) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
      hif4_decode8_even_odd<1>(c.y, l, sf2, o);
      *reinterpret_cast<uint4 *>(at + (((part + 1) ^ swz) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
      hif4_decode8_even_odd<2>(c.z, l, sf2, o);
      *reinterpret_cast<uint4 *>(at + (((part + 2) ^ swz) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
      hif4_decode8_even_odd<3>(c.w, l, sf2, o);
      *reinterpret_cast<uint4 *>(at + (((part + 3) ^ swz) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
};

// weights of 32 columns: p = 2^(s scale - ref), summed in fp32 (pairs of sums)
// and packed to bf16 for the second product, as in attend_rows_kernel; a low
// part would need columns of tensor memory that are not there, and half as
// much tensor-core work again.
__device__ __forceinline__ void weights32(const uint32_t (&s)[32], u64 scale2, u64 nref2, u64 &sum2, uint32_t *p) {
#pragma unroll
  for (int j = 0; j < 16; j++) {
    float x, y;
    upk2(fma2(pk2(__uint_as_float(s[2 * j]), __uint_as_float(s[2 * j + 1])), scale2, nref2), x, y);
    x = ex2(x);
    y = ex2(y);
    sum2 = add2(sum2, pk2(x, y));
    p[j] = pack_bf16(x, y);
  }
}

// bits 0 .. n - 1 (none for n <= 0, all for n >= 64)
__device__ __forceinline__ u64 below(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }

// Registers move from the warps that need few to the softmax: 256 x 152 +
// 256 x 64 + 128 x 40 = 60416 of the launch's 640 x 96 = 61440.
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <int DH>
__global__ void __launch_bounds__(THREADS, 1) attend_tiles_kernel(const AttendArgs a, int flip) {
  using C = Cfg<DH>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *kfull = reinterpret_cast<uint64_t *>(smem + C::BARS), *kempty = kfull + 2, *vfull = kempty + 2;
  uint64_t *vempty = vfull + 2, *sfull = vempty + 2, *pfull = sfull + 4, *odone = pfull + 4;
  uint64_t *drain = odone + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 2);
  int *found = reinterpret_cast<int *>(tmem_slot + 1);          // sequence, tile, first position
  uint8_t *hidden = reinterpret_cast<uint8_t *>(found + 3);     // [4 steps][8 blocks of 16 keys]: 1 without a page
  const CacheArgs &c = a.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kh = blockIdx.x % c.heads, split = blockIdx.y;

  // ---- which sequence and tile: the tiles of all sequences counted off, all heads of one together, the last
  // tiles first (they see the most keys; what starts last is short)
  if (warp == 0) {
    int left = blockIdx.x / c.heads, seq = -1, tile = 0, two = 1;
    for (int b0 = 0; b0 < c.B && seq < 0; b0 += 32) {
      const int b = b0 + lane;
      const int at = b < c.B ? c.cu_new[b] : 0, count = b < c.B ? c.cu_new[b + 1] - at : 0;
      // no more than the grid was sized for: the rows that are there
      const int64_t r = (int64_t)count * a.group > a.most_rows ? rows_present(a, at, count) : 0;
      const int n = (int)((r + ROWS - 1) / ROWS);
      int sum = n;
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, sum, x);
        if (lane >= x) sum += y;
      }
      const unsigned in = __ballot_sync(0xffffffffu, left < sum);
      if (in) {
        const int l = __ffs(in) - 1;
        const int upto = __shfl_sync(0xffffffffu, sum, l);
        seq = b0 + l;
        tile = upto - 1 - left;
        // 1 or 2 tiles of 128 rows
        two = __shfl_sync(0xffffffffu, r, l) - (int64_t)tile * ROWS > 128 ? 2 : 1;
      } else {
        left -= __shfl_sync(0xffffffffu, sum, 31);
      }
    }
    if (lane == 0) {
      found[0] = seq;
      found[1] = tile;
      for (int i = 0; i < 2; i++) {
        mbar_init(&kfull[i], 8);
        mbar_init(&kempty[i], two);
        mbar_init(&vfull[i], 8);
        mbar_init(&vempty[i], two);
        mbar_init(&sfull[i], 1);
        mbar_init(&sfull[2 + i], 1);
        mbar_init(&pfull[i], 4);
        mbar_init(&pfull[2 + i], 4);
        mbar_init(&odone[i], 1);
        mbar_init(&drain[i], 1);
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }
  __syncthreads();
  const int seq = found[0];
  if (seq < 0) return;
  if (warp == 8) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  const int cu0 = c.cu_new[seq], n_new = c.cu_new[seq + 1] - cu0, old = c.kv_len[seq] - n_new;
  const int64_t rows = rows_present(a, cu0, n_new), r0 = (int64_t)found[1] * ROWS;
  const int tiles_here = rows - r0 > 128 ? 2 : 1;
  const int64_t r1 = min(rows, r0 + ROWS);
  const int p_lo = old + (int)(r0 / a.group), p_top = old + (int)((r1 - 1) / a.group);
  const int64_t room = (int64_t)c.most << c.page_shift;
  int p_hi = p_top;
  if (p_hi >= room) {
    if (threadIdx.x == 0) atomicExch(c.status + 1, HIF4X_BAD_PAGE);
    p_hi = (int)(room - 1);
  }
  const KeyTiles kt(min(max(p_lo, 0), p_hi), p_hi, a.window, a.sinks, KEYS);
  const int per = (kt.n + a.sh.n - 1) / a.sh.n;
  const int first = min(kt.n, split * per), n = min(kt.n, first + per) - first;   // steps of this CTA

  // asked for where a page is none; held in a register through the loops it cost the prologue 0.6 us in spills
  if (threadIdx.x == 0) found[2] = p_lo;

  // ---- Q into shared memory (K-major panels of 64 dims, 128-byte swizzle)
  for (int e = threadIdx.x; e < tiles_here * 128 * (DH / 8); e += THREADS) {
    const int r = e / (DH / 8), q = e % (DH / 8);
    const int64_t rr = r0 + r, token = (int64_t)cu0 + rr / a.group;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (rr < r1 && token >= 0 && token < c.rows) {
      x = __ldg(reinterpret_cast<const uint4 *>(a.q + token * a.q_row + (kh * a.group + (int)(rr % a.group)) * a.q_head) + q);
      if (flip) {
        x.x ^= 0x80008000u;
        x.y ^= 0x80008000u;
        x.z ^= 0x80008000u;
        x.w ^= 0x80008000u;
      }
    }
    *reinterpret_cast<uint4 *>(smem + C::Q + (r >> 7) * C::TILE + (q >> 3) * C::PANEL + (r & 127) * 128 +
                               (((q & 7) ^ (r & 7)) << 4)) =
        make_uint4(__byte_perm(x.x, x.y, 0x5410), __byte_perm(x.z, x.w, 0x5410), __byte_perm(x.x, x.y, 0x7632),
                   __byte_perm(x.z, x.w, 0x7632));
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  if (warp >= 12) {
    // ---- decode
    regs_down<64>();
    const int w = warp - 12;
    const int *pages = c.pages + seq * c.ld_pages;
    const int last = p_hi;
    // item u: K (even) or V (odd) of step u / 2; the next one's words are on their way meanwhile, and so is what
    // the page table says of the step after
    const Loader<DH> ld(c, kh, w, lane);
    Words<DH> cur, next;
    auto key_of = [&](int i) { return kt.key0(first + i, KEYS) + w * 16; };
    auto look = [&](int i) { return i < n && key_of(i) <= last ? __ldg(pages + (key_of(i) >> c.page_shift)) : -1; };
    // an id of no page: -1, and reported where a row of this CTA would have seen the keys (steps of 128 begin before
    // the window and end behind the sinks, and pages there may have been given back)
    auto check = [&](int i, int page) {
      if (page >= 0 && page < c.num_pages) return page;
      if (lane == 0 && i < n && key_of(i) <= last) {
        const int k = key_of(i), p_first = found[2];
        if (a.window == 0 || k + 15 > p_first - a.window || k < a.sinks) atomicExch(c.status + 1, HIF4X_BAD_PAGE);
      }
      return -1;
    };
    int now = look(0), nxt = look(1);   // of the step being decoded, of the one after it
    now = check(0, now);
    if (n > 0) ld.load(cur, c.codes[0], c.meta[0], key_of(0), now);
#pragma unroll 1
    for (int u = 0; u < 2 * n; u++) {
      const int i = u >> 1, v = u & 1, s = i & 1;
      if (v == 0) {
        ld.load(next, c.codes[1], c.meta[1], key_of(i), now);
        if (lane == 0) hidden[(i & 3) * 8 + w] = now < 0 ? 1 : 0;
      } else if (i + 1 < n) {
        now = check(i + 1, nxt);
        ld.load(next, c.codes[0], c.meta[0], key_of(i + 1), now);
        nxt = look(i + 2);
      }
      if (i >= 2) ok = mbar_wait_sleep((v ? vempty : kempty) + s, ((i >> 1) - 1) & 1, c.status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      ld.store(cur, smem + (v ? C::V : C::K) + s * C::TILE);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive((v ? vfull : kfull) + s);
      cur = next;
    }
  } else if (warp >= 8) {
    // ---- both products of tile warp - 8
    regs_down<40>();
    const int t = warp - 8;
    if (t < tiles_here && n > 0 && elect_one()) {
      const uint32_t base = smem_u32(smem);
      // descriptors of the first K-substep; a step further is a constant in their address bits (16-byte units)
      const uint64_t dq = smem_desc(base + C::Q + t * C::TILE, 16u, 1024u, 2u);
      const uint64_t dk = smem_desc(base + C::K, 16u, 1024u, 2u), dv = smem_desc(base + C::V, C::PANEL, 1024u, 2u);
      const uint32_t d_s = tmem + t * 128, d_o = tmem + 256 + t * 128;
      // half step j: 64 keys, S and weights of it in half j & 1 of the tile's columns
      auto qk = [&](int j) {
        const int st = (j >> 1) & 1;
        const uint64_t k = dk + st * (C::TILE >> 4) + (j & 1) * (64 * 128 >> 4);
        if (!(j & 1)) ok = mbar_wait_sleep(&kfull[st], (j >> 2) & 1, c.status);   // both halves at once
        if (!ok) return;
        tc_fence_after();
#pragma unroll
        for (int x = 0; x < DH / 16; x++) {
          const uint32_t off = ((x >> 2) * C::PANEL + (x & 3) * 32) >> 4;
          mma_f16_ss(d_s + (j & 1) * 64, dq + off, k + off, idesc_bf16(64, 0), x > 0 ? 1u : 0u);
        }
        mma_commit(&sfull[2 * t + (j & 1)]);
        if (j & 1) mma_commit(&kempty[st]);
      };
      qk(0);
      if (ok) qk(1);
#pragma unroll 1
      for (int j = 0; j < 2 * n && ok; j++) {
        const int st = (j >> 1) & 1;
        const uint64_t v = dv + st * (C::TILE >> 4) + (j & 1) * (64 * 128 >> 4);
        if (!(j & 1)) ok = mbar_wait_sleep(&vfull[st], (j >> 2) & 1, c.status);
        ok = ok && mbar_wait_sleep(&pfull[2 * t + (j & 1)], (j >> 1) & 1, c.status);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int x = 0; x < 4; x++)
          mma_f16_ts(d_o, d_s + (j & 1) * 64 + x * 8, v + x * (2048 >> 4), idesc_bf16(DH, 1), (j > 0 || x > 0) ? 1u : 0u);
        mma_commit(&odone[t]);
        if (j & 1) mma_commit(&vempty[st]);
        if (j + 2 < 2 * n) {   // the next S of these columns, once their weights have been read
          ok = mbar_wait_sleep(&odone[t], j & 1, c.status);
          if (ok) qk(j + 2);
        }
      }
      mma_commit(&drain[t]);   // every issued product has finished before tensor memory is released
      mbar_wait_sleep(&drain[t], 0, c.status);
    }
    __syncwarp();
  } else {
    // ---- softmax: this thread's row
    regs_up<152>();
    const int t = warp >> 2;
    const int r = t * 128 + (warp & 3) * 32 + lane;
    const int64_t rr = r0 + r;
    if (t < tiles_here) {
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t ts = tmem + lanes + t * 128, to = tmem + lanes + 256 + t * 128;
      const int p = rr < r1 ? old + (int)(rr / a.group) : -1;
      // the least and the last position of this tile's rows
      const int t_lo = old + (int)((r0 + t * 128) / a.group);
      const int t_hi = old + (int)((min(r1, r0 + t * 128 + 128) - 1) / a.group);
      float ref = -INFINITY;
      u64 sum2 = pk2(0.0f, 0.0f);
#pragma unroll 1
      for (int j = 0; j < 2 * n; j++) {
        const int i = j >> 1, h = j & 1;
        ok = mbar_wait_sleep(&sfull[2 * t + h], i & 1, c.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[32], s1[32];
        tmem_ld32(ts + 64 * h, s);
        tmem_ld32(ts + 64 * h + 32, s1);
        const int key0 = kt.key0(first + i, KEYS) + 64 * h;
        const uint32_t hid = *reinterpret_cast<const uint32_t *>(hidden + (i & 3) * 8 + 4 * h);   // a byte for 16 keys
        const bool all = key0 + 63 <= t_lo && (a.window == 0 || key0 > t_hi - a.window || key0 + 63 < a.sinks) && hid == 0;
        tmem_wait_ld(s);
        tmem_loaded(s1);
        if (!all) {
          // visible columns: y <= hi and (y > lo or y < sk), 16-key blocks with a page
          const int hi = p - key0, lo = a.window ? p - a.window - key0 : -1, sk = a.sinks - key0;
          const u64 see = below(hi + 1) & (~below(lo + 1) | below(sk)) &
                          ~((hid & 1u ? 0xffffull : 0ull) | (hid & 0x100u ? 0xffffull << 16 : 0ull) |
                            (hid & 0x10000u ? 0xffffull << 32 : 0ull) | (hid & 0x1000000u ? 0xffffull << 48 : 0ull));
          const uint32_t see0 = (uint32_t)see, see1 = (uint32_t)(see >> 32);
#pragma unroll
          for (int y = 0; y < 32; y++) {
            if (!(see0 & (1u << y))) s[y] = 0xff800000u;
            if (!(see1 & (1u << y))) s1[y] = 0xff800000u;
          }
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int y = 0; y < 32; y += 4) {
          m4[0] = max3(m4[0], __uint_as_float(s[y]), __uint_as_float(s[y + 1]));
          m4[1] = max3(m4[1], __uint_as_float(s[y + 2]), __uint_as_float(s[y + 3]));
          m4[2] = max3(m4[2], __uint_as_float(s1[y]), __uint_as_float(s1[y + 1]));
          m4[3] = max3(m4[3], __uint_as_float(s1[y + 2]), __uint_as_float(s1[y + 3]));
        }
        const float m = fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]) * a.scale;
        if (__any_sync(0xffffffffu, m > ref + kLazy)) {
          const float to_ref = fmaxf(m, ref);
          const float f = ref == -INFINITY ? 0.0f : ex2(ref - to_ref);
          ref = to_ref;
          sum2 = mul2(sum2, pk2(f, f));
          if (j > 0) {   // O as of the half step before
            ok = mbar_wait_sleep(&odone[t], (j - 1) & 1, c.status);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c0 = 0; c0 < DH; c0 += 16) {
              uint32_t y[16];
              tmem_ld16(to + c0, y);
              tmem_wait_ld(y);
#pragma unroll
              for (int k = 0; k < 16; k++) y[k] = __float_as_uint(__uint_as_float(y[k]) * f);
              tmem_st16(to + c0, y);
            }
          }
        }
        const float base = ref == -INFINITY ? 0.0f : ref;
        const u64 scale2 = pk2(a.scale, a.scale), nref2 = pk2(-base, -base);
        uint32_t w[32];
        weights32(s, scale2, nref2, sum2, w);
        weights32(s1, scale2, nref2, sum2, w + 16);
        tmem_st32(ts + 64 * h, w);   // over S columns that have been read
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        // a barrier for each half: a warp may be done with the next one before another is with this one
        if (lane == 0) mbar_arrive(&pfull[2 * t + h]);
      }
      if (n > 0 && ok) {
        ok = mbar_wait_sleep(&drain[t], 0, c.status);   // all products
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      float s_even, s_odd;
      upk2(sum2, s_even, s_odd);
      const float sum = s_even + s_odd;
      const int64_t token = (int64_t)cu0 + rr / a.group;
      const bool mine = rr < r1 && token >= 0 && token < c.rows;
      const int head = kh * a.group + (int)(rr % a.group);
      const int64_t at = split * a.sh.all + token * (c.heads * a.group) + head;
      const float inv = a.sh.n > 1 ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
      if (a.sh.n > 1 && mine) a.sh.ml[at] = make_float2(ref, sum);
#pragma unroll 1
      for (int c0 = 0; c0 < DH; c0 += 32) {
        uint32_t o[32];
        __syncwarp();   // lanes of rows that are not stored are ahead
        if (n > 0) {
          tmem_ld32(to + c0, o);
          tmem_wait_ld(o);
        } else {
#pragma unroll
          for (int j = 0; j < 32; j++) o[j] = 0u;
        }
        if (!mine) continue;
        // a chunk of eight dims stands as (0 2 4 6 1 3 5 7)
        if (a.sh.n > 1) {
          float4 *dst = reinterpret_cast<float4 *>(a.sh.part + at * DH + c0);
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const int e = 8 * (j >> 1) + 2 * (j & 1);
            dst[j] = make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 4]), __uint_as_float(o[e + 1]),
                                 __uint_as_float(o[e + 5]));
          }
        } else {
          uint4 *dst = reinterpret_cast<uint4 *>(a.out + token * a.o_row + head * a.o_head + c0);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            uint32_t x[4];
#pragma unroll
            for (int k = 0; k < 4; k++)
              x[k] = sum == 0.0f ? 0u
                                 : pack_bf16(__uint_as_float(o[8 * j + k]) * inv, __uint_as_float(o[8 * j + k + 4]) * inv);
            dst[j] = make_uint4(x[0], x[1], x[2], x[3]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

}  // namespace tiles

// The shares of a (row, query head), added in their order: a CTA each, four
// warps with every fourth share and eight of them on their way at a time (the
// chain of dependent loads is the time of this kernel), joined in shared
// memory.  The sums lie by (token, query head); where both kernels ran (BOTH),
// attend_rows_kernel's are `few`, by (sequence, key head, row).  The grid then
// is one of the two: few's alone where only its sequences have shares.  In the
// other one a row of few's is known by its mark, seen when its sums have been
// read in vain: to ask before would put a load in front of every row's.

// one warp's shares: the sums of its lanes' dims and their (reference, weight)
template <int DH>
__device__ __forceinline__ float2 join_warp(const Shares &sh, int64_t at, int warp, int lane, float (&v)[DH / 32]) {
  constexpr int V = DH / 32;
  // shares s = warp, warp + 4, ... (at most 16): lane k has the k-th one's reference and weight
  const int mine = warp + 4 * lane;
  const float2 ml = mine < sh.n ? sh.ml[mine * sh.all + at] : make_float2(-INFINITY, 0.0f);
  float m = ml.x;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
  const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - m);   // nothing visible in a share: no part in the sum
  float l = f * ml.y;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
#pragma unroll
  for (int k = 0; k < V; k++) v[k] = 0.0f;
#pragma unroll 8
  for (int k = 0; k < (sh.n - warp + 3) / 4; k++) {
    const float *src = sh.part + ((warp + 4 * k) * sh.all + at) * DH + lane * V;
    const float w = __shfl_sync(0xffffffffu, f, k);
#pragma unroll
    for (int e = 0; e < V; e++) v[e] += w == 0.0f ? 0.0f : w * src[e];
  }
  return make_float2(m, l);
}

template <int DH, bool BOTH>
__global__ void __launch_bounds__(128, 16) attend_join_kernel(const AttendArgs a, const Shares few, int grid_few) {
  constexpr int V = DH / 32;
  __shared__ float so[4][DH];
  __shared__ float2 sml[4];
  const CacheArgs &c = a.c;
  const int heads = c.heads * a.group, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t at = blockIdx.x;
  int64_t token;
  int head;
  float v[V];
  float2 ml;
  if (BOTH && grid_few) {
    const int r = (int)(at % FEW_ROWS), kh = (int)(at / FEW_ROWS % c.heads), s = (int)(at / FEW_ROWS / c.heads);
    const int cu0 = c.cu_new[s], n_new = c.cu_new[s + 1] - cu0;
    if ((int64_t)n_new * a.group > FEW_ROWS || r >= rows_present(a, cu0, n_new)) return;
    token = (int64_t)cu0 + r / a.group;
    head = kh * a.group + r % a.group;
    ml = join_warp<DH>(few, at, warp, lane, v);
  } else {
    token = at / heads;
    head = (int)(at - token * heads);
    if (token < c.cu_new[0] || token >= c.cu_new[c.B]) return;   // rows of no sequence stay as they are
    const float mark = BOTH ? a.sh.ml[at].y : 0.0f;
    ml = join_warp<DH>(a.sh, at, warp, lane, v);
    if (BOTH && mark < 0.0f) {
      if (few.n == 1) return;   // its result is there already
      const int s = find_sequence(c.cu_new, c.B, token, lane & 7, 0xffu << (lane & 24)), kh = head / a.group;
      const int64_t r = (token - c.cu_new[s]) * a.group + head - kh * a.group;
      if (s >= c.B || r < 0 || r >= FEW_ROWS) return;   // a cu_new that falls: no such sums
      ml = join_warp<DH>(few, ((int64_t)s * c.heads + kh) * FEW_ROWS + r, warp, lane, v);
    }
  }
#pragma unroll
  for (int e = 0; e < V; e++) so[warp][lane * V + e] = v[e];
  if (lane == 0) sml[warp] = ml;
  __syncthreads();
  if (threadIdx.x >= DH / 2) return;
  const int d = threadIdx.x * 2;
  float top = -INFINITY, total = 0.0f, o0 = 0.0f, o1 = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; w++) top = fmaxf(top, sml[w].x);
#pragma unroll
  for (int w = 0; w < 4; w++) {
    const float g = sml[w].x == -INFINITY ? 0.0f : ex2(sml[w].x - top);
    total += g * sml[w].y;
    o0 += g * so[w][d];
    o1 += g * so[w][d + 1];
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  *reinterpret_cast<uint32_t *>(a.out + token * a.o_row + head * a.o_head + d) = pack_bf16(o0 * inv, o1 * inv);
}

// Shares of the keys of one (sequence, key head) in attend_rows_kernel.  Few
// lanes (sequence, key head): as many shares as the SMs hold CTAs at once (a
// second wave would leave most of them idle; 65536 keys of one sequence: 46 us
// in 55 shares, 61 in 27, 56 in 64).  Many: twelve CTAs for every SM, so that
// sequences of several lengths even out (64 sequences of up to 8192 keys: 168
// us in the four shares this gives, 217 unshared, 205 in twelve).  No share
// under 512 keys (eight tiles for each warp; the join is a launch of its own,
// 4 us), and no more than 2^26 partial sums (256 MB) in all.  Beside the tiles
// kernel (`both`) none under 2048: the join is then launched for sequences
// that may not be there.
static int attend_splits(int sms, int64_t lanes, int64_t keys, int64_t outputs, bool two, bool both) {
  const int64_t at_once = (two ? 2 : 3) * (int64_t)sms;
  const int64_t want = lanes * 4 <= at_once * 3 ? at_once / lanes : (12 * (int64_t)sms + lanes - 1) / lanes;
  const int64_t most = std::max<int64_t>(1, keys / (both ? 2048 : 512));
  const int64_t room = (int64_t(1) << 26) / std::max<int64_t>(1, outputs);
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, room, MOST_SPLITS}));
}

// How a call is carried out: from its sizes alone.
struct AttendPlan {
  bool rows, tiles;          // the kernels that run
  int most_rows;             // rows of a sequence up to which the first one takes it
  int grid_tiles;
  Shares sh, few;            // of the only kernel, or of the tiles kernel and (n > 0) of the rows kernel beside it
  int64_t work_bytes;
};

// Sequences of up to FEW_ROWS rows (new tokens x query heads of a key head) go
// to attend_rows_kernel, others to attend_tiles_kernel.  Only the device knows
// the lengths: where max_new allows for more rows both kernels run and each
// passes over the other's sequences, except that a single sequence is the
// tiles kernel's alone.  Each kernel has its own number of shares: a chunk's
// tiles fill the GPU by themselves, the long token beside it does not.
struct AttendSizes {
  int page_size, kv_heads, head_dim, sequences, max_pages, q_heads;
  int64_t rows;
  int window, sinks, max_new;
};

static int attend_plan(const AttendSizes &z, AttendPlan *p) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return HIF4X_ERR_LAUNCH;
  const int sms = tc::device_sms(dev);
  if (sms <= 0) return HIF4X_ERR_LAUNCH;
  const int group = z.q_heads / z.kv_heads;
  const int64_t B = z.sequences, H = z.kv_heads;
  // keys that a sequence of up to `fresh` new rows sees at most
  auto keys_of = [&](int64_t fresh) {
    const int64_t room = (int64_t)z.max_pages * z.page_size;
    return z.window > 0 ? std::min<int64_t>(room, z.window + fresh + z.sinks + 32) : room;
  };
  const int64_t keys = keys_of(z.max_new);
  p->tiles = (int64_t)z.max_new * group > 16;
  p->rows = !p->tiles || B > 1;
  p->most_rows = !p->tiles ? INT32_MAX : B > 1 ? FEW_ROWS : 0;
  p->grid_tiles = 0;
  const int64_t outs = z.rows * z.q_heads, slots = B * H * FEW_ROWS;
  p->sh.all = outs;
  p->few.n = 0;
  p->few.all = slots;
  if (p->tiles) {
    const int64_t n = z.rows * group / tiles::ROWS + B;
    if (n * H > INT32_MAX) return HIF4X_ERR_UNSUPPORTED;
    p->grid_tiles = (int)n;
    // shares of the keys: as many as fill the SMs once (sequences taken alike), four steps or more to each
    const int64_t busy = B * std::max<int64_t>(1, (z.rows * group + B * tiles::ROWS - 1) / (B * tiles::ROWS)) * H;
    p->sh.n = (int)std::max<int64_t>(
        1, std::min<int64_t>({sms / busy, keys / (4 * tiles::KEYS), (int64_t(1) << 26) / (outs * z.head_dim), MOST_SPLITS}));
    if (p->rows) p->few.n = attend_splits(sms, B * H, keys_of(FEW_ROWS), slots * z.head_dim, true, true);
  } else {
    p->sh.n = attend_splits(sms, B * H, keys, outs * z.head_dim, (int64_t)z.max_new * group > 8, false);
  }
  const int64_t sums = (p->sh.n > 1 ? p->sh.n * outs : 0) + (p->few.n > 1 ? p->few.n * slots : 0);
  p->work_bytes = sums * (4 * z.head_dim + 8);
  return HIF4X_OK;
}

// The workspace: all partial sums, then all (reference, weight) pairs.
static void place_shares(AttendPlan *p, void *work, int head_dim) {
  float *at = static_cast<float *>(work);
  for (Shares *s : {&p->sh, &p->few})
    if (s->n > 1) {
      s->part = at;
      at += s->n * s->all * head_dim;
    }
  float2 *ml = reinterpret_cast<float2 *>(at);
  for (Shares *s : {&p->sh, &p->few})
    if (s->n > 1) {
      s->ml = ml;
      ml += s->n * s->all;
    }
}

template <int DH>
static int launch_tiles(AttendArgs a, int dev, const AttendPlan &p, cudaStream_t s) {
  static tc::SharedOptIn opt_in;
  if (!opt_in(tiles::attend_tiles_kernel<DH>, tiles::Cfg<DH>::SMEM, dev)) return HIF4X_ERR_LAUNCH;
  // the kernel compares unscaled scores, so its scale is positive: a negative one turns the queries' signs
  const int flip = a.scale < 0.0f;
  a.scale = std::max(std::fabs(a.scale), 1e-35f);
  const dim3 grid((unsigned)(p.grid_tiles * a.c.heads), (unsigned)p.sh.n);
  tiles::attend_tiles_kernel<DH><<<grid, tiles::THREADS, tiles::Cfg<DH>::SMEM, s>>>(a, flip);
  HIF4X_CHECK_LAUNCH();
  return HIF4X_OK;
}

static bool attend_sizes_ok(const AttendSizes &z) {
  return z.kv_heads >= 1 && z.q_heads >= z.kv_heads && z.q_heads % z.kv_heads == 0 && z.window >= 0 && z.sinks >= 0 &&
         z.max_new >= 1 && z.window <= (1 << 30) && z.sinks <= (1 << 30) && z.rows >= 0 &&
         z.rows * z.q_heads <= INT32_MAX && z.sequences >= 1 && z.max_pages >= 1 && z.page_size >= 1 &&
         (z.head_dim == 64 || z.head_dim == 128);
}

}  // namespace hif4x

using namespace hif4x;

extern "C" int hif4x_paged_attention_work(int page_size, int kv_heads, int head_dim, int sequences, int max_pages,
                                          int q_heads, int64_t rows, int window, int sinks, int max_new,
                                          int64_t *bytes) {
  const AttendSizes z{page_size, kv_heads, head_dim, sequences, max_pages, q_heads, rows, window, sinks, max_new};
  if (!bytes || !attend_sizes_ok(z)) return HIF4X_ERR_ARG;
  *bytes = 0;
  if (rows == 0) return HIF4X_OK;
  AttendPlan p{};
  const int st = attend_plan(z, &p);
  *bytes = p.work_bytes;
  return st;
}

extern "C" int hif4x_paged_attention(const hif4x_kv_cache *kv, const hif4x_kv_batch *batch, const void *q,
                                     int64_t q_ld_row, int64_t q_ld_head, int q_heads, int64_t rows, float scale,
                                     int window, int sinks, int max_new, void *out, int64_t o_ld_row,
                                     int64_t o_ld_head, void *work, int64_t work_bytes, void *stream) {
  AttendArgs a{};
  int st = cache_args(kv, batch, rows, &a.c);
  if (st != HIF4X_OK) return st;
  const AttendSizes z{kv->page_size, kv->kv_heads, kv->head_dim, batch->sequences, batch->max_pages, q_heads,
                      rows, window, sinks, max_new};
  if (!attend_sizes_ok(z)) return HIF4X_ERR_ARG;
  if (rows == 0) return HIF4X_OK;
  if (!q || !out || q == out) return HIF4X_ERR_ARG;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u) || q_ld_row % 8 || q_ld_head % 8 ||
      o_ld_row % 8 || o_ld_head % 8)
    return HIF4X_ERR_ARG;
  AttendPlan p{};
  st = attend_plan(z, &p);
  if (st != HIF4X_OK) return st;
  if (p.work_bytes > 0 && (!work || work_bytes < p.work_bytes || (reinterpret_cast<uintptr_t>(work) & 15u)))
    return HIF4X_ERR_ARG;
  a.q = static_cast<const __nv_bfloat16 *>(q);
  a.q_row = q_ld_row;
  a.q_head = q_ld_head;
  a.out = static_cast<__nv_bfloat16 *>(out);
  a.o_row = o_ld_row;
  a.o_head = o_ld_head;
  a.group = q_heads / kv->kv_heads;
  a.scale = scale * 1.4426950408889634f;
  a.window = window;
  a.sinks = sinks;
  place_shares(&p, work, kv->head_dim);
  a.sh = p.sh;
  a.most_rows = p.most_rows;
  cudaStream_t s = (cudaStream_t)stream;
  if (p.tiles) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return HIF4X_ERR_LAUNCH;
    st = kv->head_dim == 128 ? launch_tiles<128>(a, dev, p, s) : launch_tiles<64>(a, dev, p, s);
    if (st != HIF4X_OK) return st;
  }
  if (p.rows) {
    AttendArgs r = a;
    if (p.tiles) {
      r.sh = p.few;
      r.slots = 1;
      r.mark = p.sh.n > 1 ? p.sh.ml : nullptr;
    }
    const dim3 grid((unsigned)batch->sequences, (unsigned)kv->kv_heads, (unsigned)r.sh.n);
    const bool two = (int64_t)max_new * a.group > 8;
    if (kv->head_dim == 128) {
      if (two) attend_rows_kernel<128, 2><<<grid, 128, 0, s>>>(r);
      else attend_rows_kernel<128, 1><<<grid, 128, 0, s>>>(r);
    } else {
      if (two) attend_rows_kernel<64, 2><<<grid, 128, 0, s>>>(r);
      else attend_rows_kernel<64, 1><<<grid, 128, 0, s>>>(r);
    }
    HIF4X_CHECK_LAUNCH();
  }
  if (p.sh.n > 1 || p.few.n > 1) {
    const int grid_few = p.sh.n == 1;
    const unsigned blocks = (unsigned)(grid_few ? p.few.all : p.sh.all);
    if (p.few.n > 0) {
      if (kv->head_dim == 128) attend_join_kernel<128, true><<<blocks, 128, 0, s>>>(a, p.few, grid_few);
      else attend_join_kernel<64, true><<<blocks, 128, 0, s>>>(a, p.few, grid_few);
    } else {
      if (kv->head_dim == 128) attend_join_kernel<128, false><<<blocks, 128, 0, s>>>(a, p.few, 0);
      else attend_join_kernel<64, false><<<blocks, 128, 0, s>>>(a, p.few, 0);
    }
    HIF4X_CHECK_LAUNCH();
  }
  return HIF4X_OK;
}
