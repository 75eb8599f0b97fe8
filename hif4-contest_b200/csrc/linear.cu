// linear.cu -- y = act(x W^T + bias) + residual with W in packed HiF4, on the
// sm_100a tensor cores.
//
// A HiF4 value is a bf16 number (hif4_bits.cuh), so W is decoded to bf16 and
// multiplied by the bf16 activations with fp32 sums: nothing is lost before
// the one rounding of the result.  W travels packed (4.5 bit) and is decoded
// next to the multiply: few rows are bound by W's bytes, many by the tensor
// cores.
//
// A CTA computes 128 rows of W (the M side) x NT rows of x (the N side, 16 to
// 256) over its share of C:
//   warp 0   one lane brings x tiles (NT x 64) by TMA, 128-byte swizzle
//   warp 1   one lane issues tcgen05.mma kind::f16 (M 128, N NT, K 16)
//   warp 2   one lane brings W's codes by TMA, 128 rows x 256 elements (16 KB)
//   warps 4-19  four warpgroups decode the 64-element steps in turn: a thread
//            is one row of W, reads its 32 bytes and one meta word, and writes
//            32 columns of bf16 pairs to tensor memory, where the MMA reads A
//            from.  (A decoding warp alone issues an instruction in 5 to 6
//            cycles: with two warps a scheduler a step took 830 cycles, with
//            four 600, of which the ALU pipe is busy for 350.)  W's tile never
//            passes shared memory as bf16: that leaves shared memory's
//            bandwidth to x alone (a 128 x 256 x 64 step would otherwise write
//            and read 96 KB there, more than its MMA time).
// C is shared out over a cluster of up to 4 CTAs where the tiles alone do not
// fill the GPU; the partial sums meet through distributed shared memory and
// are added in rank order, so results do not depend on timing.
// Every wait is bounded (sm100.cuh); on expiry the kernel records
// HIF4X_TIMEOUT and ends.
#include <algorithm>

#include "common.cuh"
#include "hif4_bits.cuh"
#include "sm100.cuh"

namespace hif4x {
namespace lin {

using namespace tc;

constexpr int STAGES = 4;        // 64-element steps of x and of decoded W in flight
constexpr int CODE_STAGES = 3;   // 256-element boxes of packed W in flight
constexpr int CODE_BYTES = 128 * 128;
constexpr int THREADS = 640;
constexpr int BM = 128;
constexpr int MOST_RANKS = 4;    // CTAs of a cluster that share a tile's C (clusters of 8 do not fit every GPC twice)

struct Args {
  int64_t T, N;
  int nb, nt, per;          // 64-groups of C; x rows of a tile; groups of a cluster rank (a multiple of 4)
  const uint32_t *meta;
  const void *bias;
  int bias_bf16, act;
  const uint16_t *res;
  int64_t ldr;
  uint16_t *y;
  int64_t ldy;
  int vec;                  // rows of y and residual take 16-byte accesses
  uint32_t tmem_cols;
  int *status;
};

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// 1 / (1 + exp(-z)) without a sum that cancels or an exponential out of range:
// a few steps of its own size on both sides of zero.
__device__ __forceinline__ float sigmoid(float z) {
  const float e = expf(-fabsf(z));
  return (z < 0.0f ? e : 1.0f) / (1.0f + e);
}

__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case HIF4X_ACT_RELU: return v > 0.0f ? v : (v != v ? v : 0.0f);
    case HIF4X_ACT_GELU: return v * normcdff(v);
    case HIF4X_ACT_GELU_TANH:   // (1 + tanh(z)) / 2 = 1 / (1 + exp(-2z))
      return v * sigmoid(2.0f * 0.7978845608028654f * (v + 0.044715f * v * v * v));
    case HIF4X_ACT_SILU: return v * sigmoid(v);
    default: return v;
  }
}

__global__ void __launch_bounds__(THREADS) linear_kernel(const __grid_constant__ CUtensorMap map_x,
                                                         const __grid_constant__ CUtensorMap map_w, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int x_bytes = a.nt * 128;
  uint8_t *sx = smem, *sw = smem + STAGES * x_bytes;
  uint64_t *full_x = reinterpret_cast<uint64_t *>(sw + CODE_STAGES * CODE_BYTES);
  uint64_t *full_a = full_x + STAGES, *empty = full_a + STAGES, *full_w = empty + STAGES;
  uint64_t *empty_w = full_w + CODE_STAGES, *done = empty_w + CODE_STAGES;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row0 = (int64_t)blockIdx.x * BM, tok0 = (int64_t)blockIdx.y * a.nt;
  const int ranks = gridDim.z, rank = blockIdx.z;
  const int k0 = min(a.nb, rank * a.per), steps = min(a.nb, k0 + a.per) - k0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      mbar_init(&full_x[s], 1);
      mbar_init(&full_a[s], 4);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < CODE_STAGES; s++) {
      mbar_init(&full_w[s], 1);
      mbar_init(&empty_w[s], 16);
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(a.tmem_cols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_a = *tmem_slot, tmem_d = tmem_a + STAGES * 32;   // A stages, then the accumulator
  bool ok = true;

  if (warp == 0) {
    if (elect_one()) {
      int i = 0;
      for (; i < steps; i++) {
        const int s = i % STAGES;
        if (i >= STAGES) ok = mbar_wait_sleep(&empty[s], ((i / STAGES) - 1) & 1, a.status);
        if (!ok) break;
        mbar_expect_tx(&full_x[s], x_bytes);
        tma_load_2d(&map_x, sx + s * x_bytes, &full_x[s], (k0 + i) * 64, (int)tok0);
      }
      // no copy may be in flight when the CTA ends
      for (int s = 0; s < STAGES; s++)
        if (i > s) mbar_wait_sleep(&full_x[s], ((i - 1 - s) / STAGES) & 1, a.status);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = idesc_bf16((uint32_t)a.nt, 0);
      const uint64_t dx = smem_desc(smem_u32(sx), 16u, 1024u, 2u);   // + 2 for 32 bytes further
      for (int i = 0; i < steps; i++) {
        const int s = i % STAGES, ph = (i / STAGES) & 1;
        ok = mbar_wait_sleep(&full_x[s], ph, a.status) &&
             mbar_wait_sleep(&full_a[s], ph, a.status);
        if (!ok) break;
        tc_fence_after();
        const uint64_t x = dx + (uint32_t)(s * x_bytes >> 4);
#pragma unroll
        for (int j = 0; j < 4; j++)
          mma_f16_ts(tmem_d, tmem_a + s * 32 + j * 8, x + 2 * j, idesc, (i > 0 || j > 0) ? 1u : 0u);
        mma_commit(&empty[s]);
      }
      mma_commit(done);
    }
  } else if (warp == 2) {
    if (elect_one()) {
      const int boxes = (steps + 3) / 4;
      int i = 0;
      for (; i < boxes; i++) {
        const int s = i % CODE_STAGES;
        if (i >= CODE_STAGES) ok = mbar_wait_sleep(&empty_w[s], ((i / CODE_STAGES) - 1) & 1, a.status);
        if (!ok) break;
        mbar_expect_tx(&full_w[s], CODE_BYTES);
        tma_load_2d(&map_w, sw + s * CODE_BYTES, &full_w[s], (k0 + 4 * i) * 32, (int)row0);
      }
      for (int s = 0; s < CODE_STAGES; s++)
        if (i > s) mbar_wait_sleep(&full_w[s], ((i - 1 - s) / CODE_STAGES) & 1, a.status);
    }
  } else if (warp >= 4) {
    // ---- decode: thread = row of W (tensor memory lane); warpgroup g has group g of every box, stage g
    const int g = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;
    const int64_t row = row0 + r;
    const uint32_t *meta = a.meta + (row < a.N ? row : 0) * a.nb + k0 + g;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    // 16-byte chunk c of row r lies at chunk c ^ (r & 7)
    const uint8_t *src0 = sw + r * 128 + (((2 * g) ^ (r & 7)) << 4), *src1 = sw + r * 128 + (((2 * g + 1) ^ (r & 7)) << 4);
    const int boxes = (steps + 3) / 4, mine = (steps - g + 3) / 4;   // this warpgroup's steps: the first boxes
    uint32_t m = mine > 0 ? __ldg(meta) : 0u;
    int cs = 0, cp = 0;   // code stage and its phase
    for (int b = 0; b < boxes && ok; b++) {
      const uint32_t next = b + 1 < mine ? __ldg(meta + 4 * (b + 1)) : 0u;
      ok = mbar_wait_sleep(&full_w[cs], cp, a.status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint4 c0 = *reinterpret_cast<const uint4 *>(src0 + cs * CODE_BYTES);
      const uint4 c1 = *reinterpret_cast<const uint4 *>(src1 + cs * CODE_BYTES);
      if (b < mine) {
        const uint32_t w[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
        uint32_t v[32];
        hif4_decode64(w, m, v);
        if (b > 0) {
          ok = mbar_wait_sleep(&empty[g], (b - 1) & 1, a.status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
        }
        tmem_st32(tmem_a + lanes + g * 32, v);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full_a[g]);
      }
      // the box is given back here, where the decoding has used every lane's words: behind their loads alone, the
      // next box could overwrite words still on their way
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_w[cs]);
      if (++cs == CODE_STAGES) {
        cs = 0;
        cp ^= 1;
      }
      m = next;
    }
    // ---- the accumulator to shared memory, [x row][row of W], over the x stages
    ok = mbar_wait_sleep(done, 0, a.status);
    __syncwarp();
    tc_fence_after();
    float *part = reinterpret_cast<float *>(sx);
    for (int n = g * 16; n < a.nt; n += 64) {
      uint32_t d[16];
      if (steps > 0) {
        tmem_ld16(tmem_d + lanes + n, d);
        tmem_wait_ld(d);
      } else {
#pragma unroll
        for (int k = 0; k < 16; k++) d[k] = 0u;
      }
#pragma unroll
      for (int k = 0; k < 16; k++) part[(n + k) * BM + r] = __uint_as_float(d[k]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_a), "r"(a.tmem_cols));
  }
  if (ranks > 1) cluster_sync();
  // ---- the ranks' sums, bias, activation, residual: 8 outputs of one x row a thread
  const uint32_t base = smem_u32(sx);
  const int rows_here = (int)min((int64_t)a.nt, a.T - tok0);
  for (int e = threadIdx.x; e < ((rows_here - rank + ranks - 1) / ranks) * (BM / 8); e += THREADS) {
    const int t = (e / (BM / 8)) * ranks + rank, c = (e % (BM / 8)) * 8;
    const int64_t n = row0 + c;
    if (n >= a.N) continue;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const uint32_t at = base + (uint32_t)(t * BM + c) * 4u;
    const int64_t tok = tok0 + t;
    const int m = (int)min((int64_t)8, a.N - n);
    const bool wide = a.vec && m == 8;
    uint4 res = make_uint4(0, 0, 0, 0);   // on its way while the sums are read
    if (wide && a.res != nullptr) res = *reinterpret_cast<const uint4 *>(a.res + tok * a.ldr + n);
    float4 p[MOST_RANKS], q[MOST_RANKS];
#pragma unroll
    for (int z = 0; z < MOST_RANKS; z++)
      if (z < ranks) {
        const uint32_t from = ranks > 1 ? mapa(at, z) : at;
        p[z] = ld_cluster4(from);
        q[z] = ld_cluster4(from + 16);
      }
#pragma unroll
    for (int z = 0; z < MOST_RANKS; z++)
      if (z < ranks) {
        v[0] += p[z].x; v[1] += p[z].y; v[2] += p[z].z; v[3] += p[z].w;
        v[4] += q[z].x; v[5] += q[z].y; v[6] += q[z].z; v[7] += q[z].w;
      }
    if (a.bias != nullptr) {
#pragma unroll
      for (int k = 0; k < 8; k++)
        if (k < m)
          v[k] += a.bias_bf16 ? bf16_bits_to_f32(static_cast<const uint16_t *>(a.bias)[n + k])
                              : static_cast<const float *>(a.bias)[n + k];
    }
    if (a.act != HIF4X_ACT_NONE) {
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] = activate(v[k], a.act);
    }
    uint16_t *dst = a.y + tok * a.ldy + n;
    if (wide) {
      if (a.res != nullptr) {
        const uint32_t w[4] = {res.x, res.y, res.z, res.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
          v[2 * k] += __uint_as_float(w[k] << 16);
          v[2 * k + 1] += __uint_as_float(w[k] & 0xffff0000u);
        }
      }
      uint32_t o[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
        o[k] = *reinterpret_cast<const uint32_t *>(&b);
      }
      *reinterpret_cast<uint4 *>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; k++)
        if (k < m) {
          if (a.res != nullptr) v[k] += bf16_bits_to_f32(a.res[tok * a.ldr + n + k]);
          dst[k] = __bfloat16_as_ushort(__float2bfloat16_rn(v[k]));
        }
    }
  }
  if (ranks > 1) cluster_sync();   // no CTA leaves while another reads its sums
}

// Tensor map of rows of `inner` bytes or bf16 values, boxes of `box` x `box_rows`, 128-byte swizzle.
static bool map_rows(CUtensorMap *map, CUtensorMapDataType type, const void *base, int64_t inner, int64_t outer,
                     int64_t pitch_bytes, int box, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
  cuuint64_t strides[1] = {(cuuint64_t)pitch_bytes};
  cuuint32_t boxes[2] = {(cuuint32_t)box, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, type, 2, const_cast<void *>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int smem_bytes(int nt) {
  return STAGES * nt * 128 + CODE_STAGES * CODE_BYTES + (3 * STAGES + 2 * CODE_STAGES + 1) * 8 + 16 + 1024;
}

}  // namespace lin
}  // namespace hif4x

using namespace hif4x;

extern "C" int hif4x_linear_packed(const void *x, int64_t ldx, const uint32_t *meta, const uint8_t *codes, int64_t T,
                                   int64_t N, int64_t C, const void *bias, int bias_dtype, int act,
                                   const void *residual, int64_t ldr, void *y, int64_t ldy, void *stream) {
  using namespace lin;
  if (T < 0 || N < 1 || C < 64 || C % 64 || act < HIF4X_ACT_NONE || act > HIF4X_ACT_SILU) return HIF4X_ERR_ARG;
  if (T == 0) return HIF4X_OK;
  if (!x || !meta || !codes || !y || ldx < C || ldx % 8 || ldy < N || (residual && ldr < N)) return HIF4X_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(codes)) & 15u) return HIF4X_ERR_ARG;
  if (bias && bias_dtype != HIF4X_DT_F32 && bias_dtype != HIF4X_DT_BF16) return HIF4X_ERR_ARG;
  if (T > INT32_MAX - 256 || N > INT32_MAX - 256 || C > (1 << 30)) return HIF4X_ERR_UNSUPPORTED;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return HIF4X_ERR_LAUNCH;
  const int sms = device_sms(dev);
  if (sms <= 0 || dev >= kMaxDevices) return HIF4X_ERR_LAUNCH;
  static SharedOptIn opt_in;
  Args a{};
  a.status = status_words(dev);
  if (!opt_in(linear_kernel, smem_bytes(256), dev) || !a.status) return HIF4X_ERR_LAUNCH;

  const int64_t tiles_n = (N + BM - 1) / BM;
  // x rows of a tile: as few tiles as hold them, all alike.  A step's decoding takes 600 cycles whatever its rows and
  // shared memory 2.25 a row (x in and out), 576 at 256: tiles of fewer rows only add steps.
  int64_t tiles_t = (T + 255) / 256;
  a.nt = (int)(((T + tiles_t - 1) / tiles_t + 15) / 16 * 16);
  tiles_t = (T + a.nt - 1) / a.nt;
  if (tiles_t > 65535) return HIF4X_ERR_UNSUPPORTED;
  a.nb = (int)(C / 64);
  // share C out while that gives more SMs a CTA; boxes of 4 steps stay whole, so the last CTA may have fewer than the
  // others, but none has nothing (C = 1088: 8, 8 and 1 steps)
  int ranks = 1;
  while (ranks < MOST_RANKS && tiles_n * tiles_t * ranks * 2 <= sms && a.nb >= 8 * ranks) ranks *= 2;
  a.per = (int)(((a.nb + ranks - 1) / ranks + 3) / 4 * 4);
  ranks = (a.nb + a.per - 1) / a.per;
  a.T = T;
  a.N = N;
  a.meta = meta;
  a.bias = bias;
  a.bias_bf16 = bias_dtype == HIF4X_DT_BF16;
  a.act = act;
  a.res = static_cast<const uint16_t *>(residual);
  a.ldr = ldr;
  a.y = static_cast<uint16_t *>(y);
  a.ldy = ldy;
  a.vec = (reinterpret_cast<uintptr_t>(y) & 15u) == 0 && ldy % 8 == 0 &&
          (!residual || ((reinterpret_cast<uintptr_t>(residual) & 15u) == 0 && ldr % 8 == 0));
  a.tmem_cols = a.nt <= 128 ? 256u : 512u;
  CUtensorMap mx, mw;
  if (!map_rows(&mx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, x, C, T, ldx * 2, 64, a.nt) ||
      !map_rows(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, C / 2, N, C / 2, 128, BM))
    return HIF4X_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)tiles_n, (unsigned)tiles_t, (unsigned)ranks);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem_bytes(a.nt);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 1;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = (unsigned)ranks;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, linear_kernel, mx, mw, a) != cudaSuccess) {
    cudaGetLastError();
    return HIF4X_ERR_LAUNCH;
  }
  return HIF4X_OK;
}
