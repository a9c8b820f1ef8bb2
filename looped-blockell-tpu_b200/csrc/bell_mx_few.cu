// bell_mx_few.cu — the MXFP4 linear and gated feed-forward for few tokens (up
// to BELL_MX_FEW_ROWS), where launches and latency are the time: one launch for
// the whole operator, quantisation of the rows included.
//
// The same sums as bell_mx.cu.  A scale block's dot product is an integer: the
// e2m1 grid doubled is 0, 1, 2, 3, 4, 6, 8, 12, so
//   sum_i x_i w_i = (sx sw / 4) * sum_i (2x_i)(2w_i),
// and one int8 mma.sync m16n8k32 (k = 32 = the scale block) gives the exact
// sums of 16 outputs x 8 tokens, scaled and added in fp32 in a fixed order.
// The 128-row tcgen05 tile would compute 128 tokens for one, and its pipeline
// of barriers, TMEM and bulk copies takes longer to start than these products
// take (measured beside the dispatch rule below).
//
// A job is 32 outputs (a quarter or half of a block-row; gated: 32 gate and
// the same 32 up outputs, one scale block of h).  The eight warps of a CTA
// share a job's live slots; a warp quantises the rows of its slot's columns
// into its own shared memory, converts the weights' nibbles in registers and
// multiplies; the warps' sums meet in shared memory, in warp order.
//
// The gated operator is one cooperative kernel: after the h of all jobs the
// grid meets at a barrier and goes on with the down projection's jobs.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <string>

#include "bell_mx.cuh"
#include "bell_mx_gemm.h"

namespace bell {
namespace mx {
namespace few {

static constexpr int kWarps = 8;
static constexpr int kThr = 32 * kWarps;

// Where a phase's rows come from.
enum Source : int32_t { kBf16 = 0, kF32 = 1, kChunks = 2 };

struct Phase {
  const void* src;
  int64_t ld;
  Source kind;
  int32_t R, K0, K1;
  int32_t C;  // column blocks of the rows
  const uint8_t *w0, *w1;
  Plan p0, p1;
};

struct Args {
  int32_t T;
  Phase first, second;  // gate/up and down, or the linear alone
  uint8_t* h;
  __nv_bfloat16 *gate, *up;
  void* out;
  const void* residual;
  int32_t out_f32;
};

// Eight nibbles to eight doubled int8 values: a holds values 0..3, b 4..7.
// prmt looks four nibbles up in a table of eight bytes; bit 3 of a selector
// nibble (the code's sign) replicates the looked-up byte's sign bit instead, 0
// for these magnitudes.  So the word itself yields the non-negative values and
// zeros; the negated magnitudes of the rest are looked up without the sign and
// kept where it is set.
__device__ __forceinline__ void expand(uint32_t w, uint32_t& a, uint32_t& b) {
  const uint32_t m = w & 0x77777777u, s = (w >> 3) & 0x11111111u;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(a) : "r"(0x03020100u), "r"(0x0C080604u), "r"(w));
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(b) : "r"(0x03020100u), "r"(0x0C080604u), "r"(w >> 16));
  a |= __byte_perm(0xFDFEFF00u, 0xF4F8FAFCu, m) & __byte_perm(0xFF00u, 0u, s);
  b |= __byte_perm(0xFDFEFF00u, 0xF4F8FAFCu, m >> 16) & __byte_perm(0xFF00u, 0u, s >> 16);
}

__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}

// A warp's rows of one slot: [token][B] doubled int8 values and the blocks'
// scales / 4.  Rows of B + 16 bytes spread the banks.
template <int B, int NG>
struct alignas(16) Rows {
  static constexpr int LD = B + 16;
  int8_t v[NG * 8][LD];
  float s[NG * 8][B / kBlock];
};

template <int B, int NG>
struct alignas(16) Shared {
  union {
    Rows<B, NG> rows[kWarps];
    float sums[kWarps][NG * 8][32];  // [warp][token][output] of one matrix
  };
};

// Quantise (or fetch quantised) the rows' columns of block c.
template <int B, int NG>
__device__ __forceinline__ void put_rows(const Phase& ph, int T, int groups, int c, Rows<B, NG>& to) {
  constexpr int BLOCKS = B / kBlock;
  const int lane = threadIdx.x & 31;
  for (int i = lane; i < groups * 8 * BLOCKS; i += 32) {
    const int t = i / BLOCKS, j = i % BLOCKS;
    uint4 q = make_uint4(0u, 0u, 0u, 0u);
    uint32_t byte = 127u;
    if (t < T) {
      if (ph.kind == kChunks) {
        const uint8_t* ch = static_cast<const uint8_t*>(ph.src) + int64_t(c) * row_chunk(B);
        q = ld_global_v4(ch + code_off(t, j, kRows * 32));  // not through the read-only path: h is this kernel's
        byte = *static_cast<const volatile uint8_t*>(ch + kRows * B / 2 + scale_off(t, j));
      } else {
        float v[32];
        const int64_t at = t * ph.ld + int64_t(c) * B + j * kBlock;
        if (ph.kind == kF32)
          load32(static_cast<const float*>(ph.src) + at, v);
        else
          load32(static_cast<const __nv_bfloat16*>(ph.src) + at, v);
        q = quantize32(v, byte);
      }
    }
    uint32_t e[8];
    expand(q.x, e[0], e[1]);
    expand(q.y, e[2], e[3]);
    expand(q.z, e[4], e[5]);
    expand(q.w, e[6], e[7]);
    *reinterpret_cast<uint4*>(&to.v[t][j * kBlock]) = make_uint4(e[0], e[1], e[2], e[3]);
    *reinterpret_cast<uint4*>(&to.v[t][j * kBlock + 16]) = make_uint4(e[4], e[5], e[6], e[7]);
    to.s[t][j] = 0.25f * scale_value(byte);
  }
}

// acc += the products of one slot: outputs [32 part, 32 part + 32) of a tile.
// Fragment k order: lane l % 4 owns word l % 4 of a block's 16 bytes, its first
// four values as k = 4 (l % 4).. and the others as 16 + 4 (l % 4).., the same in
// both operands.
template <int B, int NG>
__device__ __forceinline__ void slot_product(const uint8_t* tile, int part, const Rows<B, NG>& x, int groups,
                                             float (&acc)[NG][2][4]) {
  constexpr int BLOCKS = B / kBlock;
  const int lane = threadIdx.x & 31, row = lane >> 2, word = lane & 3;
  uint32_t w[BLOCKS][4];  // [block][row group of 8]
  uint32_t sc[4];         // the four scale bytes of this lane's row in each group
#pragma unroll
  for (int j = 0; j < BLOCKS; ++j)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      w[j][g] = __ldg(reinterpret_cast<const unsigned*>(tile + code_off(part * 32 + g * 8 + row, j, B * 32)) + word);
#pragma unroll
  for (int g = 0; g < 4; ++g)
    sc[g] = __ldg(reinterpret_cast<const unsigned*>(tile + B * B / 2 + scale_off(part * 32 + g * 8 + row, 0)));
#pragma unroll
  for (int j = 0; j < BLOCKS; ++j) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t a[4];
      expand(w[j][half * 2], a[0], a[2]);
      expand(w[j][half * 2 + 1], a[1], a[3]);
      const float s0 = scale_value((sc[half * 2] >> (8 * j)) & 255u), s1 = scale_value((sc[half * 2 + 1] >> (8 * j)) & 255u);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        if (g < groups) {
          const uint2 b = *reinterpret_cast<const uint2*>(&x.v[g * 8 + row][j * kBlock + word * 8]);
          int d[4];
          mma_s8(d, a, b.x, b.y);
          const float t0 = x.s[g * 8 + word * 2][j], t1 = x.s[g * 8 + word * 2 + 1][j];
          // (d s) t: a product of the scales alone could overflow next to d = 0
          acc[g][half][0] = fmaf(float(d[0]) * s0, t0, acc[g][half][0]);
          acc[g][half][1] = fmaf(float(d[1]) * s0, t1, acc[g][half][1]);
          acc[g][half][2] = fmaf(float(d[2]) * s1, t0, acc[g][half][2]);
          acc[g][half][3] = fmaf(float(d[3]) * s1, t1, acc[g][half][3]);
        }
      }
    }
  }
}

// The sums of one job's 32 outputs of one or two matrices: sum[m][k] is token
// warp + 8 k, output `lane`.
template <int B, int NG, int MATS>
__device__ __forceinline__ void job_sums(const Phase& ph, int T, int job, Shared<B, NG>& sh, float (&sum)[MATS][NG]) {
  constexpr int PARTS = B / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = job / PARTS, part = job % PARTS, groups = (T + 7) / 8;
  const int n0 = __ldg(ph.p0.counts + r), n1 = MATS == 2 ? __ldg(ph.p1.counts + r) : 0;
  float acc[MATS][NG][2][4];
#pragma unroll
  for (int m = 0; m < MATS; ++m)
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[m][g][i >> 2][i & 3] = 0.f;
  // the warps take the live slots of the first matrix in turn, then the second's
#pragma unroll
  for (int m = 0; m < MATS; ++m) {
    const int K = m ? ph.K1 : ph.K0, n = m ? n1 : n0;
    const uint32_t* entries = (m ? ph.p1 : ph.p0).entries + int64_t(r) * K;
    const uint8_t* w = (m ? ph.w1 : ph.w0) + int64_t(r) * K * tile_chunk(B);
    for (int i = m ? (warp + kWarps - n0 % kWarps) % kWarps : warp; i < n; i += kWarps) {
      const uint32_t e = __ldg(entries + i);
      put_rows<B, NG>(ph, T, groups, int(e & 0xFFFFu), sh.rows[warp]);
      __syncwarp();
      slot_product<B, NG>(w + int64_t(e >> 16) * tile_chunk(B), part, sh.rows[warp], groups, acc[m]);
      __syncwarp();
    }
  }
  const int row = lane >> 2, col = (lane & 3) * 2;
#pragma unroll
  for (int m = 0; m < MATS; ++m) {
    __syncthreads();  // the sums take the rows' place, and the other matrix's
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        sh.sums[warp][g * 8 + col + (i & 1)][(i >> 2) * 16 + ((i >> 1) & 1) * 8 + row] = acc[m][g][i >> 2][i & 3];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      sum[m][k] = 0.f;
#pragma unroll
      for (int v = 0; v < kWarps; ++v) sum[m][k] += sh.sums[v][warp + 8 * k][lane];
    }
  }
  __syncthreads();  // read before the next job's rows
}

template <int B, int NG>
__device__ void gated_jobs(const Args& a, Shared<B, NG>& sh) {
  constexpr int PARTS = B / 32;
  const Phase& ph = a.first;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int job = blockIdx.x; job < ph.R * PARTS; job += gridDim.x) {
    float sum[2][NG];
    job_sums<B, NG, 2>(ph, a.T, job, sh, sum);
    const int r = job / PARTS, part = job % PARTS;
#pragma unroll
    for (int k = 0; k < NG; ++k) {  // a lane per feature: one scale block of h
      const int t = warp + 8 * k;
      if (t >= a.T) break;
      const float g = sum[0][k], u = sum[1][k];
      if (a.gate) {
        const int64_t at = int64_t(t) * ph.R * B + int64_t(r) * B + part * 32 + lane;
        a.gate[at] = __float2bfloat16_rn(g);
        a.up[at] = __float2bfloat16_rn(u);
      }
      const float2 h2 = silu_mul2(make_float2(g, g), make_float2(u, u));
      const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(h2.x) & 0x7FFFFFFFu);  // NaN on top
      const uint32_t byte = scale_byte(top);
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = h2.x * scale_inverse(byte);
      uint32_t code = (pack_e2m1(v) & 15u) << (4 * (lane & 7));  // this lane's nibble of its word
      code |= __shfl_xor_sync(0xffffffffu, code, 1);
      code |= __shfl_xor_sync(0xffffffffu, code, 2);
      code |= __shfl_xor_sync(0xffffffffu, code, 4);
      uint8_t* ch = a.h + int64_t(r) * row_chunk(B);
      if ((lane & 7) == 0)
        *reinterpret_cast<uint32_t*>(ch + code_off(t, part, kRows * 32) + (lane >> 3) * 4) = code;
      if (lane == 0) ch[kRows * B / 2 + scale_off(t, part)] = uint8_t(byte);
    }
  }
}

template <int B, int NG>
__device__ void linear_jobs(const Args& a, const Phase& ph, Shared<B, NG>& sh) {
  constexpr int PARTS = B / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int job = blockIdx.x; job < ph.R * PARTS; job += gridDim.x) {
    float sum[1][NG];
    job_sums<B, NG, 1>(ph, a.T, job, sh, sum);
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const int t = warp + 8 * k;
      if (t >= a.T) break;
      const int64_t at = int64_t(t) * ph.R * B + int64_t(job) * 32 + lane;
      float v = sum[0][k];
      if (a.out_f32) {
        if (a.residual) v += static_cast<const float*>(a.residual)[at];
        static_cast<float*>(a.out)[at] = v;
      } else {
        if (a.residual) v += __bfloat162float(static_cast<const __nv_bfloat16*>(a.residual)[at]);
        static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
      }
    }
  }
}

template <int B, int NG>
__global__ void __launch_bounds__(kThr, 2) bell_mx_few_linear_kernel(const Args a) {
  __shared__ Shared<B, NG> sh;
  linear_jobs<B, NG>(a, a.first, sh);
}

template <int B, int NG>
__global__ void __launch_bounds__(kThr, 2) bell_mx_few_swiglu_kernel(const Args a) {
  __shared__ Shared<B, NG> sh;
  gated_jobs<B, NG>(a, sh);
  cooperative_groups::this_grid().sync();
  linear_jobs<B, NG>(a, a.second, sh);
}

template <int B, int NG>
static int launch(const Args& a, bool gated, int32_t max_ctas, cudaStream_t s) {
  int dev = 0, sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(BELL_ERR_LAUNCH, "cudaGetDevice");
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(kThr);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  cfg.attrs = attr;
  const int jobs = a.first.R * (B / 32);
  if (max_ctas <= 0) max_ctas = jobs;
  cudaError_t e;
  if (gated) {
    // every CTA must be resident at the grid's barrier
    static std::atomic<int> resident[64];
    auto kern = bell_mx_few_swiglu_kernel<B, NG>;
    int n = resident[dev].load();
    if (!n) {
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, kThr, 0) != cudaSuccess || n < 1)
        return fail(BELL_ERR_LAUNCH, "MXFP4 kernel for few rows: no CTA fits");
      resident[dev].store(n);
    }
    cfg.gridDim = dim3(unsigned(std::min({jobs, n * sms, max_ctas})));
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kern, a);
  } else {
    cfg.gridDim = dim3(unsigned(std::min(jobs, max_ctas)));
    e = cudaLaunchKernelEx(&cfg, bell_mx_few_linear_kernel<B, NG>, a);
  }
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(BELL_ERR_LAUNCH, std::string("MXFP4 kernel for few rows: ") + cudaGetErrorString(e));
  }
  return BELL_OK;
}

static Phase phase(const RowSource& x, const BellMxEll& w0, const BellMxEll* w1) {
  Phase ph{};
  ph.src = x.chunks ? x.chunks : x.src;
  ph.ld = x.ld;
  ph.kind = x.chunks ? kChunks : x.f32 ? kF32 : kBf16;
  ph.R = w0.R;
  ph.C = w0.C;
  ph.K0 = w0.K;
  ph.w0 = static_cast<const uint8_t*>(w0.chunks);
  ph.p0 = plan_of(w0.plan, w0.R, w0.K);
  if (w1) {
    ph.K1 = w1->K;
    ph.w1 = static_cast<const uint8_t*>(w1->chunks);
    ph.p1 = plan_of(w1->plan, w1->R, w1->K);
  }
  return ph;
}

static int go(const Args& a, int32_t B, bool gated, int32_t max_ctas, cudaStream_t s) {
  if (B == 128) return a.T <= 8 ? launch<128, 1>(a, gated, max_ctas, s) : launch<128, 4>(a, gated, max_ctas, s);
  return a.T <= 8 ? launch<64, 1>(a, gated, max_ctas, s) : launch<64, 4>(a, gated, max_ctas, s);
}

}  // namespace few

int few_linear(int64_t T, const RowSource& x, const BellMxEll& w, const void* residual, void* out, int32_t out_f32,
               int32_t max_ctas, cudaStream_t s) {
  few::Args a{};
  a.T = int32_t(T);
  a.first = few::phase(x, w, nullptr);
  a.out = out;
  a.residual = residual;
  a.out_f32 = out_f32;
  return few::go(a, w.B, false, max_ctas, s);
}

int few_swiglu(int64_t T, const RowSource& x, const BellMxEll& g, const BellMxEll& u, const BellMxEll& w, void* h,
               void* gate_pre, void* up_out, const void* residual, void* out, int32_t out_f32, int32_t max_ctas,
               cudaStream_t s) {
  few::Args a{};
  a.T = int32_t(T);
  a.first = few::phase(x, g, &u);
  RowSource hs{};
  hs.chunks = h;
  a.second = few::phase(hs, w, nullptr);
  a.h = static_cast<uint8_t*>(h);
  a.gate = static_cast<__nv_bfloat16*>(gate_pre);
  a.up = static_cast<__nv_bfloat16*>(up_out);
  a.out = out;
  a.residual = residual;
  a.out_f32 = out_f32;
  return few::go(a, w.B, true, max_ctas, s);
}

}  // namespace mx
}  // namespace bell
