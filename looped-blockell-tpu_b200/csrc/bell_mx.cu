// bell_mx.cu — Block-ELL products of MXFP4 rows and tiles on tcgen05
// (kind::mxf4: e2m1 operands, one ue8m0 scale for 32 values, fp32 sums): the
// linear, and the gated feed-forward's gate and up projections with SiLU*up
// and the re-quantisation of h in the epilogue.
//
// y[t, rB + o] = sum over live slots k of row r, i < B, of
//                Q(x)[t, c(r,k) B + i] Q(W)[r, k, i, o]
//
// A job is one accumulator: 128 tokens x one block-row of one matrix.  A unit
// is one job (linear) or a gate job and an up job (gated).  A slot of a job
// takes one activation chunk and one weight chunk (codes and scales, bulk
// copies; layouts in bell_mx.cuh); its scale images are copied into TMEM and
// B/64 MMAs of 128 x B x 64 issued.  A pipeline stage holds up to SLOTS slots
// of a job, and a job takes ceil(K / SLOTS) stages whatever its live slots (a
// dead row's are empty), so that every warp knows the order of the stages
// without reading the plan first.
//
// The issuing warp's wait, commit and bookkeeping cost about 300 cycles a
// stage, more than a slot's MMAs (B = 128: 128 cycles at the fp4 rate).  Hence
// the multi-slot stages, and two issuers: job j of the CTA belongs to issuer
// j & 1 (gated: gate jobs and up jobs), each with a ring of its own.
//
// Warps: 0-3 producers (ring w / 2; stage use h of a ring belongs to its
// producer h & 1), 4-19 epilogue (a warp takes the TMEM lane quadrant w % 4 and
// one 32-column block of a unit; at B = 64, two blocks, two groups of eight
// warps take the CTA's units in turn), 20 and 21 issuers (20 owns TMEM).
// Accumulators form a ring of ACCS in job order, so the issuers run ahead of the
// epilogue.  The TMEM scale
// columns belong to the stage: a stage is refilled only after its MMAs have
// completed, so the scales of MMAs in flight are never overwritten.
// Token-major, because a lane of the epilogue then holds 32 consecutive
// features of its token: one scale block, quantised without talking to another
// lane and stored as 16 bytes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <string>

#include "bell_mx.cuh"

namespace bell {
namespace mx {

static constexpr int kProducers = 4;  // two to a ring
static constexpr int kEpiWarps = 16;
static constexpr int kIssuer = kProducers + kEpiWarps;  // 20, 21
static constexpr int kThreads = 32 * (kIssuer + 2);

template <int B>
struct Geo {
  static constexpr int A = row_chunk(B), W = tile_chunk(B);
  static constexpr int SLOT = A + W;             // 17408 / 7168 bytes, multiples of 256
  static constexpr int SLOTS = B == 128 ? 2 : 4;
  static constexpr int STAGE = SLOTS * SLOT;
  static constexpr int NR = B == 128 ? 3 : 4;    // stages of a ring
  static constexpr int NS = 2 * NR;
  static constexpr int ACCS = B == 128 ? 3 : 4;
  static constexpr int SF_COL = ACCS * B;        // 8 scale columns per slot of a stage from here
  static constexpr int SMEM = NS * STAGE + 1024 + 1024;
  // a producer's wait for the release of use h - NR must not meet the parity of
  // use h - 2 NR: that one is released before h - 2 - NR, which it waited for
  static_assert(NR > 2, "mbarrier parity");
  static_assert(SF_COL + NS * SLOTS * 8 <= 512, "TMEM columns");
  static_assert(SMEM <= 232448, "shared memory");
};

struct Params {
  int64_t T;
  int32_t mtiles, R, C, K0, K1;
  const uint8_t* x;               // rows of chunks, C column blocks
  const uint8_t *w0, *w1;         // tiles
  Plan p0, p1;
  uint8_t* h;                     // gated: [mtiles, R] chunks
  __nv_bfloat16 *gate, *up;       // gated, optional [T, R*B]
  void* out;                      // linear [T, R*B]
  const void* residual;           // linear, optional, out's type
  int32_t out_f32;
  int32_t* status;
  uint64_t timeout_ns;
};

struct Smem {
  uint8_t* stages;
  uint64_t *full, *empty, *acc_full, *acc_empty, *drain;
  uint32_t *count, *tmem_slot;  // live slots of each stage
  volatile int* abort_flag;
};

template <int B>
__device__ __forceinline__ Smem carve(uint8_t* raw) {
  using G = Geo<B>;
  Smem s;
  s.stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ctl = s.stages + G::NS * G::STAGE;
  s.full = reinterpret_cast<uint64_t*>(ctl);
  s.empty = s.full + G::NS;
  s.acc_full = s.empty + G::NS;
  s.acc_empty = s.acc_full + G::ACCS;
  s.drain = s.acc_empty + G::ACCS;
  s.count = reinterpret_cast<uint32_t*>(s.drain + 2);
  s.tmem_slot = s.count + G::NS;
  s.abort_flag = reinterpret_cast<volatile int*>(s.tmem_slot + 1);
  return s;
}

// The CTA's units are blockIdx.x + i * gridDim.x; ring k's job i is unit i of
// matrix k (gated) or unit 2i + k (linear).
template <bool GATED>
__device__ __forceinline__ int ring_jobs(const Params& p, int k) {
  const int units = p.mtiles * p.R, first = int(blockIdx.x), grid = int(gridDim.x);
  const int mine = first < units ? (units - first + grid - 1) / grid : 0;
  return GATED ? mine : (mine - k + 1) / 2;
}
template <bool GATED>
__device__ __forceinline__ int job_unit(int i, int k) {
  return int(blockIdx.x) + (GATED ? i : 2 * i + k) * int(gridDim.x);
}

// ---------------------------------------------------------------- producer

template <int B, bool GATED>
__device__ void produce(const Params& p, const Smem& s, int ring, int sub, const Ctl& ctl) {
  using G = Geo<B>;
  const int lane = threadIdx.x & 31;
  const uint64_t keep = policy_evict_last(), pass = policy_evict_normal();
  const int mat = GATED ? ring : 0;
  const int K = mat ? p.K1 : p.K0;
  const uint8_t* w = mat ? p.w1 : p.w0;
  const uint32_t* entries = (mat ? p.p1 : p.p0).entries;
  const int per_job = (K + G::SLOTS - 1) / G::SLOTS;
  const int jobs = ring_jobs<GATED>(p, ring);
  uint64_t* full = s.full + ring * G::NR;
  uint64_t* empty = s.empty + ring * G::NR;
  int job = sub / per_job, part = sub % per_job;  // of the next use
  int m = 0, r = 0;
  // this producer's next use's entries travel while the one before is issued
  auto fetch = [&]() -> uint32_t {
    const int u = job_unit<GATED>(job, ring);
    m = u / p.R;
    r = u - m * p.R;
    const int k = part * G::SLOTS + lane;
    return lane < G::SLOTS && k < K ? __ldg(entries + int64_t(r) * K + k) : kNoSlot;
  };
  uint32_t e_next = job < jobs ? fetch() : kNoSlot;
  uint32_t stage = uint32_t(sub), phase = 0;
  bool ok = true;
  int64_t filled = 0;
  while (job < jobs) {
    const uint32_t e = e_next;
    const uint8_t* xm = p.x + int64_t(m) * p.C * G::A;
    const uint8_t* wr = w + int64_t(r) * K * G::W;
    part += 2;
    while (part >= per_job) {
      part -= per_job;
      ++job;
    }
    if (job < jobs) e_next = fetch();
    ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1u, ctl));
    if (!ok) break;
    const int cnt = __popc(__ballot_sync(0xffffffffu, e != kNoSlot));
    uint8_t* st = s.stages + (ring * G::NR + int(stage)) * G::STAGE;
    uint32_t ent[G::SLOTS];
#pragma unroll
    for (int i = 0; i < G::SLOTS; ++i) ent[i] = __shfl_sync(0xffffffffu, e, i);
    if (elect_one()) {
      s.count[ring * G::NR + stage] = uint32_t(cnt);
      if (cnt)
        mbar_arrive_expect_tx(&full[stage], uint32_t(cnt) * uint32_t(G::SLOT));
      else
        mbar_arrive(&full[stage]);
#pragma unroll
      for (int i = 0; i < G::SLOTS; ++i) {
        if (i < cnt) {
          bulk_load(st + i * G::SLOT, xm + int64_t(ent[i] & 0xFFFFu) * G::A, G::A, &full[stage], pass);
          bulk_load(st + i * G::SLOT + G::A, wr + int64_t(ent[i] >> 16) * G::W, G::W, &full[stage], keep);
        }
      }
    }
    __syncwarp();
    ++filled;
    stage += 2;
    if (stage >= uint32_t(G::NR)) {
      stage -= G::NR;
      phase ^= 1u;
    }
  }
  if (!ok && lane == 0) {  // let this producer's copies land before the CTA exits (bounded)
    for (int i = 0; i < G::NR && filled > 0; ++i, --filled) {
      if (stage < 2u) {
        stage += G::NR;
        phase ^= 1u;
      }
      stage -= 2;
      const uint32_t a = smem_u32(&full[stage]);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(a, phase) && globaltimer_ns() - t0 < 100000000ull) {
      }
    }
  }
}

// ------------------------------------------------------------------ issuer

template <int B, bool GATED>
__device__ void issue(const Params& p, const Smem& s, uint32_t tmem, int ring, const Ctl& ctl) {
  using G = Geo<B>;
  const bool leader = elect_one();
  const uint32_t a0 = sdesc_lo(smem_u32(s.stages) + ring * (G::NR * G::STAGE), 128);
  const uint32_t sf0 = sdesc_lo(smem_u32(s.stages) + ring * (G::NR * G::STAGE), 16);
  const int K = GATED && ring ? p.K1 : p.K0;
  const int per_job = (K + G::SLOTS - 1) / G::SLOTS;
  const int jobs = ring_jobs<GATED>(p, ring);
  uint64_t* full = s.full + ring * G::NR;
  uint64_t* empty = s.empty + ring * G::NR;
  uint32_t stage = 0, phase = 0;
  uint32_t acc = uint32_t(ring), use = 0;  // job 2i + ring of the CTA: accumulator (2i + ring) % ACCS
  bool ok = true;
  for (int i = 0; i < jobs && ok; ++i) {
    ok = __all_sync(0xffffffffu, mbar_wait(&s.acc_empty[acc], (use & 1u) ^ 1u, ctl));
    if (!ok) break;
    tc_fence_after();
    const uint32_t d = tmem + acc * B;
    uint32_t more = 0;
    for (int part = 0; part < per_job; ++part) {
      ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, ctl));
      if (!ok) break;
      tc_fence_after();
      const int n = int(s.count[ring * G::NR + stage]);
      if (leader) {
        const uint32_t st = stage * uint32_t(G::STAGE >> 4);
        const uint32_t sf = tmem + G::SF_COL + (ring * G::NR + stage) * (G::SLOTS * 8);
#pragma unroll
        for (int j = 0; j < G::SLOTS; ++j) {
          if (j < n) {
            const uint32_t at = st + j * (G::SLOT >> 4);
            copy_scales(sf + j * 8, sf0 + at + ((G::A - kScaleBytes) >> 4));
            copy_scales(sf + j * 8 + 4, sf0 + at + ((G::SLOT - kScaleBytes) >> 4));
#pragma unroll
            for (int kk = 0; kk < B / 64; ++kk)
              mma_mxf4(d, a0 + at + kk * (kRows * 32 >> 4), a0 + at + ((G::A + kk * B * 32) >> 4),
                       idesc_mxf4(kRows, B, kk * 2), sf + j * 8, sf + j * 8 + 4, j > 0 || kk > 0 ? 1u : more);
          }
        }
        mma_commit(&empty[stage]);
      }
      __syncwarp();
      more = 1;
      if (++stage == G::NR) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (!ok) break;
    if (leader) mma_commit(&s.acc_full[acc]);
    __syncwarp();
    acc += 2;
    if (acc >= uint32_t(G::ACCS)) {
      acc -= G::ACCS;
      ++use;
    }
  }
  if (leader) {  // every MMA has completed before TMEM is released
    mma_commit(&s.drain[ring]);
    const uint32_t a = smem_u32(&s.drain[ring]);
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(a, 0) && globaltimer_ns() - t0 < 100000000ull) {
    }
  }
  __syncwarp();
}

// ---------------------------------------------------------------- epilogue

// h = silu(g) u = g u / (1 + e^-g) in fp32, two at a time (about 1e-6
// relative): the hardware tanh form of the bf16 kernels (2^-11) would move one
// in a few hundred of h's 4-bit codes to a neighbour.  Subnormal intermediates
// are flushed: e^-g below 2^-126 next to 1, and 1 / (1 + e^-g) below 2^-126.
__device__ __forceinline__ float2 silu_mul2(float2 g, float2 u) {
  const float2 t = mul2(g, make_float2(-1.4426950408889634f, -1.4426950408889634f));
  float2 e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
  const float2 a = add2(e, make_float2(1.f, 1.f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(a.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(a.y));
  return mul2(mul2(g, r), u);
}

template <int B, bool GATED>
__device__ void epilogue(const Params& p, const Smem& s, uint32_t tmem, const Ctl& ctl) {
  using G = Geo<B>;
  constexpr int NB = B / 32;             // scale blocks (32 features) of a unit
  constexpr int GROUPS = kEpiWarps / (4 * NB);
  constexpr int JOBS = GATED ? 2 : 1;
  const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) - kProducers;
  const int q = w & 3, j = (w >> 2) % NB, group = (w >> 2) / NB;
  const int units = p.mtiles * p.R;
  const int64_t ld = int64_t(p.R) * B;
  const uint32_t lanes = uint32_t(q * 32) << 16;
  const int step = GROUPS * int(gridDim.x);
  uint32_t acc = uint32_t(group * JOBS), use = 0;  // accumulator of this unit's first job
  int c0 = 0, c1 = 0;  // live slots of the next unit's rows, read a unit ahead
  auto counts = [&](int u) {
    c0 = __ldg(p.p0.counts + u % p.R);
    if (GATED) c1 = __ldg(p.p1.counts + u % p.R);
  };
  int u = int(blockIdx.x) + group * int(gridDim.x);
  if (u < units) counts(u);
  for (; u < units; u += step) {
    const int m = u / p.R, r = u - m * p.R;
    const int n = q * 32 + lane;
    const int64_t t = int64_t(m) * kRows + n;
    const bool live0 = c0 > 0, live1 = c1 > 0;
    if (u + step < units) counts(u + step);
    const int64_t at = t * ld + int64_t(r) * B + j * 32;
    if constexpr (GATED) {
      const uint32_t a0 = acc, a1 = acc + 1 == uint32_t(G::ACCS) ? 0u : acc + 1;
      const uint32_t use1 = a1 ? use : use + 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&s.acc_full[a0], use & 1u, ctl))) return;
      if (!__all_sync(0xffffffffu, mbar_wait(&s.acc_full[a1], use1 & 1u, ctl))) return;
      tc_fence_after();
      float h[32];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t col = tmem + lanes + uint32_t(j * 32 + half * 16);
        uint32_t gr[16], ur[16];
        tmem_ld16x2_sync(col + a0 * B, gr, col + a1 * B, ur);
        if (half) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&s.acc_empty[a0]);
            mbar_arrive(&s.acc_empty[a1]);
          }
        }
        if (!live0 || !live1) {  // a projection without a live slot is zero
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (!live0) gr[i] = 0u;
            if (!live1) ur[i] = 0u;
          }
        }
        if (p.gate && t < p.T) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t a[4], c[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              a[e] = pack_bf16x2(__uint_as_float(gr[8 * i + 2 * e]), __uint_as_float(gr[8 * i + 2 * e + 1]));
              c[e] = pack_bf16x2(__uint_as_float(ur[8 * i + 2 * e]), __uint_as_float(ur[8 * i + 2 * e + 1]));
            }
            st_global_v4(p.gate + at + half * 16 + 8 * i, a[0], a[1], a[2], a[3]);
            st_global_v4(p.up + at + half * 16 + 8 * i, c[0], c[1], c[2], c[3]);
          }
        }
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float2 v = silu_mul2(make_float2(__uint_as_float(gr[i]), __uint_as_float(gr[i + 1])),
                                     make_float2(__uint_as_float(ur[i]), __uint_as_float(ur[i + 1])));
          h[half * 16 + i] = v.x;
          h[half * 16 + i + 1] = v.y;
        }
      }
      uint32_t byte;
      const uint4 c = quantize32(h, byte);
      if (t < p.T) {
        uint8_t* ch = p.h + (int64_t(m) * p.R + r) * G::A;
        st_global_v4(ch + code_off(n, j, kRows * 32), c.x, c.y, c.z, c.w);
        ch[kRows * B / 2 + scale_off(n, j)] = uint8_t(byte);
      }
    } else {
      if (!__all_sync(0xffffffffu, mbar_wait(&s.acc_full[acc], use & 1u, ctl))) return;
      tc_fence_after();
      uint32_t a[32];
      tmem_ld32_sync(tmem + lanes + acc * B + j * 32, a);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.acc_empty[acc]);
      if (t < p.T) {
        float f[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = live0 ? __uint_as_float(a[i]) : 0.f;
        if (p.out_f32) {
          float* o = static_cast<float*>(p.out) + at;
          const float* rs = static_cast<const float*>(p.residual);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (rs) {
              const uint4 v = ld_global_v4(rs + at + 4 * i);
              f[4 * i] += __uint_as_float(v.x);
              f[4 * i + 1] += __uint_as_float(v.y);
              f[4 * i + 2] += __uint_as_float(v.z);
              f[4 * i + 3] += __uint_as_float(v.w);
            }
            st_global_v4(o + 4 * i, __float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]),
                         __float_as_uint(f[4 * i + 2]), __float_as_uint(f[4 * i + 3]));
          }
        } else {
          __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + at;
          const __nv_bfloat16* rs = static_cast<const __nv_bfloat16*>(p.residual);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (rs) {
              const uint4 v = ld_global_v4(rs + at + 8 * i);
              const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 x2 = unpack_bf16x2(vw[e]);
                f[8 * i + 2 * e] += x2.x;
                f[8 * i + 2 * e + 1] += x2.y;
              }
            }
            st_global_v4(o + 8 * i, pack_bf16x2(f[8 * i], f[8 * i + 1]), pack_bf16x2(f[8 * i + 2], f[8 * i + 3]),
                         pack_bf16x2(f[8 * i + 4], f[8 * i + 5]), pack_bf16x2(f[8 * i + 6], f[8 * i + 7]));
          }
        }
      }
    }
    acc += GROUPS * JOBS;
    while (acc >= uint32_t(G::ACCS)) {
      acc -= G::ACCS;
      ++use;
    }
  }
}

template <int B, bool GATED>
__global__ void __launch_bounds__(kThreads, 1) bell_mx_kernel(const Params p) {
  using G = Geo<B>;
  extern __shared__ uint8_t smem_raw[];
  const Smem s = carve<B>(smem_raw);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < G::NS; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < G::ACCS; ++i) {
      mbar_init(&s.acc_full[i], 1);
      mbar_init(&s.acc_empty[i], B / 32 * 4);  // the epilogue warps of a unit
    }
    mbar_init(&s.drain[0], 1);
    mbar_init(&s.drain[1], 1);
    *s.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kIssuer) {
    tmem_alloc(s.tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s.tmem_slot;
  const Ctl ctl{s.abort_flag, p.status, p.timeout_ns};
  griddep_launch();
  griddep_wait();  // the rows come from the kernel before
  if (warp < kProducers)
    produce<B, GATED>(p, s, warp >> 1, warp & 1, ctl);
  else if (warp < kIssuer)
    epilogue<B, GATED>(p, s, tmem, ctl);
  else
    issue<B, GATED>(p, s, tmem, warp - kIssuer, ctl);
  tc_fence_before();
  __syncthreads();
  if (warp == kIssuer) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int B, bool GATED>
static int launch(const Params& p, int32_t max_ctas, bool dependent, cudaStream_t s) {
  auto kern = bell_mx_kernel<B, GATED>;
  if (int rc = set_smem(reinterpret_cast<const void*>(kern), Geo<B>::SMEM)) return rc;
  int sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  int64_t grid = int64_t(p.mtiles) * p.R;
  if (grid > sms) grid = sms;
  if (max_ctas > 0 && grid > max_ctas) grid = max_ctas;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Geo<B>::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(BELL_ERR_LAUNCH, std::string("MXFP4 kernel: ") + cudaGetErrorString(e));
  }
  return BELL_OK;
}

static int check_ell(const BellMxEll& e, const char* name) {
  if (!e.chunks || !e.plan) return fail(BELL_ERR_ARG, std::string(name) + ": NULL chunks/plan");
  if (e.B != 64 && e.B != 128) return fail(BELL_ERR_SHAPE, std::string(name) + ": tile size B must be 64 or 128");
  if (e.R < 1 || e.C < 1 || e.K < 1 || e.R > (1 << 23) || e.C > 65535 || e.K > 65535)
    return fail(BELL_ERR_SHAPE, std::string(name) + ": R, C, K must be >= 1, R <= 2^23 and C, K <= 65535");
  if (!aligned16(e.chunks) || !aligned16(e.plan))
    return fail(BELL_ERR_ALIGN, std::string(name) + ": chunks and plan must be 16-byte aligned");
  return BELL_OK;
}

static int check_size(int64_t T, int32_t R) {
  if (T < 0 || T > (int64_t(1) << 31) - 256) return fail(BELL_ERR_SHAPE, "T must be in [0, 2^31 - 256)");
  if ((T + kRows - 1) / kRows * R > INT_MAX / 4) return fail(BELL_ERR_SHAPE, "T x block-rows too large");
  return BELL_OK;
}

static Params base_params(int64_t T, const BellMxEll& w0, const BellMxEll* w1, const void* x, int32_t* status) {
  Params p{};
  p.T = T;
  p.mtiles = int32_t((T + kRows - 1) / kRows);
  p.R = w0.R;
  p.C = w0.C;
  p.K0 = w0.K;
  p.x = static_cast<const uint8_t*>(x);
  p.w0 = static_cast<const uint8_t*>(w0.chunks);
  p.p0 = plan_of(w0.plan, w0.R, w0.K);
  if (w1) {
    p.K1 = w1->K;
    p.w1 = static_cast<const uint8_t*>(w1->chunks);
    p.p1 = plan_of(w1->plan, w1->R, w1->K);
  }
  p.status = status;
  p.timeout_ns = wait_budget_ns();
  return p;
}

// Quantise the caller's rows first where it gave any.
template <class D>
static int quantize_source(const D* d, const BellMxEll& w, void* stream) {
  if (!d->x_src) return BELL_OK;
  return bell_mx_quantize_rows(d->T, w.C * w.B, w.B, d->src_dtype, d->x_src, d->ld_src, d->x, stream);
}

static int linear(int64_t T, const void* x, const BellMxEll& w, const void* residual, void* out, int32_t out_dtype,
                  int32_t max_ctas, int32_t* status, bool dependent, cudaStream_t s) {
  Params p = base_params(T, w, nullptr, x, status);
  p.out = out;
  p.residual = residual;
  p.out_f32 = out_dtype == BELL_DTYPE_F32;
  return w.B == 128 ? launch<128, false>(p, max_ctas, dependent, s) : launch<64, false>(p, max_ctas, dependent, s);
}

}  // namespace mx
}  // namespace bell

using namespace bell;

extern "C" {

int bell_linear_mx(const BellMxLinearDesc* d, void* stream) {
  if (!d) return fail(BELL_ERR_ARG, "descriptor is NULL");
  if (int rc = mx::check_ell(d->w, "weight")) return rc;
  if (int rc = mx::check_size(d->T, d->w.R)) return rc;
  if (d->out_dtype != BELL_DTYPE_BF16 && d->out_dtype != BELL_DTYPE_F32)
    return fail(BELL_ERR_DTYPE, "out_dtype must be bf16 or f32");
  if (d->T > 0 && (!d->x || !d->out)) return fail(BELL_ERR_ARG, "x and out must be non-NULL");
  if (!aligned16(d->x) || !aligned16(d->out) || !aligned16(d->residual))
    return fail(BELL_ERR_ALIGN, "x, out and residual must be 16-byte aligned");
  if (d->max_ctas < 0) return fail(BELL_ERR_ARG, "max_ctas must be >= 0");
  if (int rc = require_sm100()) return rc;
  if (d->T == 0) return BELL_OK;
  int32_t* status = d->status ? d->status : default_status_ptr();
  if (!status) return BELL_ERR_LAUNCH;
  if (int rc = mx::quantize_source(d, d->w, stream)) return rc;
  return mx::linear(d->T, d->x, d->w, d->residual, d->out, d->out_dtype, d->max_ctas, status, true,
                    static_cast<cudaStream_t>(stream));
}

int bell_swiglu_fwd_mx(const BellMxFFNDesc* d, void* stream) {
  if (!d) return fail(BELL_ERR_ARG, "descriptor is NULL");
  if (int rc = mx::check_ell(d->gate, "gate")) return rc;
  if (int rc = mx::check_ell(d->up, "up")) return rc;
  if (int rc = mx::check_ell(d->down, "down")) return rc;
  const BellMxEll &g = d->gate, &u = d->up, &w = d->down;
  if (g.B != u.B || g.B != w.B) return fail(BELL_ERR_SHAPE, "gate, up and down must share the tile size");
  if (g.R != u.R || g.C != u.C) return fail(BELL_ERR_SHAPE, "gate and up must have the same R and C");
  if (w.C != g.R || w.R != g.C) return fail(BELL_ERR_SHAPE, "down must map d_ff back to d_model");
  if (int rc = mx::check_size(d->T, g.R > w.R ? g.R : w.R)) return rc;
  if (d->out_dtype != BELL_DTYPE_BF16 && d->out_dtype != BELL_DTYPE_F32)
    return fail(BELL_ERR_DTYPE, "out_dtype must be bf16 or f32");
  if (d->T > 0 && (!d->x || !d->h || !d->out)) return fail(BELL_ERR_ARG, "x, h and out must be non-NULL");
  if (!d->gate_pre != !d->up_out) return fail(BELL_ERR_ARG, "gate_pre and up_out come together");
  if (!aligned16(d->x) || !aligned16(d->h) || !aligned16(d->out) || !aligned16(d->residual) ||
      !aligned16(d->gate_pre) || !aligned16(d->up_out))
    return fail(BELL_ERR_ALIGN, "buffers must be 16-byte aligned");
  if (d->max_ctas < 0) return fail(BELL_ERR_ARG, "max_ctas must be >= 0");
  if (int rc = require_sm100()) return rc;
  if (d->T == 0) return BELL_OK;
  int32_t* status = d->status ? d->status : default_status_ptr();
  if (!status) return BELL_ERR_LAUNCH;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int rc = mx::quantize_source(d, g, stream)) return rc;
  mx::Params p = mx::base_params(d->T, g, &u, d->x, status);
  p.h = static_cast<uint8_t*>(d->h);
  p.gate = static_cast<__nv_bfloat16*>(d->gate_pre);
  p.up = static_cast<__nv_bfloat16*>(d->up_out);
  if (int rc = g.B == 128 ? mx::launch<128, true>(p, d->max_ctas, true, s) : mx::launch<64, true>(p, d->max_ctas, true, s))
    return rc;
  return mx::linear(d->T, d->h, w, d->residual, d->out, d->out_dtype, d->max_ctas, status, true, s);
}

}  // extern "C"
