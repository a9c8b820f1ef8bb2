// bell_mx.cu — Block-ELL products of MXFP4 rows and tiles on tcgen05
// (kind::mxf4: e2m1 operands, one ue8m0 scale for 32 values, fp32 sums): the
// linear, and the gated feed-forward's gate and up projections with SiLU*up
// and the re-quantisation of h in the epilogue.
//
// y[t, rB + o] = sum over live slots k of row r, i < B, of
//                Q(x)[t, c(r,k) B + i] Q(W)[r, k, i, o]
//
// The backward of the gated part is the same kernel with another epilogue: it
// computes the projections g and u again, exactly as the forward had them, and
// turns d_h into d_gate and d_up.  That costs the products a second time and
// saves keeping g and u: in bf16 their writes cost 74 us of the forward's 289
// at T = 8192, d = 4096, d_ff = 16384, their reads as much in the backward, and
// their rounding was a third of the tile gradients' error.
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
// The issuing warp's wait, commit and bookkeeping cost about 170 cycles a
// stage, as much as a slot's MMAs (B = 128: 120 cycles and 20 for its scales).
// Hence the multi-slot stages, and two issuers: job j of the CTA belongs to
// issuer j & 1 (gated: gate jobs and up jobs), each with a ring of its own.
//
// A linear with units enough takes two token tiles to a unit (kPairs): one ring,
// whose stages hold the rows of both tiles and the weights once, and issuer k
// takes tile k from every stage; a stage is free when both have committed it, so
// neither is more than the ring ahead of the other.  At B = 128 13 KB for a tile's
// slot instead of 17.4 (16384 -> 4096 at T = 16384 148 -> 133 us), at B = 64 fewer
// stages too (2048 -> 8192, 84 -> 72 us).  The gated kernel gains nothing that way
// (313 us with a tile, 322 with two): two gates and two ups need four
// accumulators and TMEM holds three, so the next unit's gates wait for most of an
// epilogue.
//
// What bounds it: B = 128, the way from the L2 into the SM, 60 bytes a cycle, and
// the ring's latency.  Of the linear's 133 us (4.2 PFLOP/s) the copies and the
// epilogue without MMAs take 102, the MMAs and the epilogue without copies 102,
// the MMAs alone 76 (120 cycles a slot; its scales 20), copies and MMAs without
// the output 109.  B = 64, gated: the epilogue's latency, a chain of 16
// instructions an output in 16 warps (T = 16384, d = 2048, d_ff = 8192: 125 us;
// without the SiLU's exponential and reciprocal 104); issue slots are busy for
// 56 % of the time, the special functions 59 %, the tensor pipe 15 %.
//
// Warps: 0-5 producers (ring w / 3; stage use h of a ring belongs to its producer
// h % 3; kPairs leaves 3-5 idle), 6-21 epilogue (a warp takes the TMEM lane
// quadrant warp % 4 and one 32-column block of a unit; at B = 64, two blocks, two
// groups of eight warps take the CTA's units in turn), 22 and 23 issuers (22 owns
// TMEM).  A producer's turn, from a stage's release to its copies' issue, is on
// the ring's path: with one tile to a unit 156 us with one producer a ring, 147
// with two or three; gated B = 64 128 us with two, 125 with three.  Accumulators
// form a ring of ACCS in job order, so the issuers run ahead of the epilogue.
//
// Few units (a linear of few tokens with long rows): split mode.  A cluster of
// `split` CTAs shares one unit, each ring of each CTA takes an equal range of the
// stages into an accumulator of its own, and the partial sums meet in distributed
// shared memory, in a fixed order.
//
// The TMEM scale columns belong to the stage: a stage is refilled only after its
// MMAs have completed, so the scales of MMAs in flight are never overwritten.
// Token-major, because a lane of the epilogue then holds 32 consecutive features
// of its token: one scale block, quantised without talking to another lane and
// stored as 16 bytes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <string>

#include "bell_mx.cuh"

namespace bell {
namespace mx {

static constexpr int kProducers = 6;
static constexpr int kEpiWarps = 16;
static constexpr int kIssuer = kProducers + kEpiWarps;  // 22, 23
static constexpr int kThreads = 32 * (kIssuer + 2);
static constexpr int kMaxSplit = 8;  // CTAs that share a unit: the portable cluster

// What a kernel's epilogue does with its accumulators; kPairs: a linear whose
// two issuers take two token tiles of one unit from one ring.
enum Mode : int { kLinear, kPairs, kGated, kGatedBackward };

template <int B, Mode MODE>
struct Geo {
  static constexpr bool GATED = MODE == kGated || MODE == kGatedBackward, PAIRS = MODE == kPairs;
  static constexpr int A = row_chunk(B), W = tile_chunk(B);
  static constexpr int TILES = PAIRS ? 2 : 1;    // token tiles of a unit
  static constexpr int SLOT = TILES * A + W;     // 17408 / 7168 / 26112 bytes, multiples of 256
  static constexpr int SLOTS = B == 128 ? 2 : 4;
  static constexpr int STAGE = SLOTS * SLOT;
  static constexpr int RINGS = PAIRS ? 1 : 2;
  static constexpr int NR = B == 64 || PAIRS ? 4 : 3;  // stages of a ring
  static constexpr int NS = RINGS * NR;
  static constexpr int PER = kProducers / 2;      // producers of a ring
  static constexpr int ACCS = B == 128 ? 3 : 4;
  // TMEM: the accumulators, then 8 scale columns for each slot that an issuer
  // takes from a stage
  static constexpr int SF_COL = ACCS * B, SF_STAGE = SLOTS * 8;
  static constexpr int SMEM = NS * STAGE + 1024 + 1024;
  // a producer's wait for the release of use h - NR must not meet the parity of
  // use h - 2 NR: that one is released no later than h - PER - NR, which it
  // waited for
  static_assert(NR >= PER && RINGS * PER <= kProducers, "mbarrier parity");
  static_assert(SF_COL + 2 * NR * SF_STAGE <= 512, "TMEM columns");
  static_assert(SMEM <= 232448, "shared memory");
};

struct Params {
  int64_t T;
  int32_t mtiles, R, C, K0, K1;
  const uint8_t* x;               // rows of chunks, C column blocks
  const void* src;                // or, x null: T <= BELL_MX_DIRECT_ROWS rows, quantised here
  int64_t ld_src;
  int32_t src_f32;
  const uint8_t *w0, *w1;         // tiles
  Plan p0, p1;
  uint8_t* h;                     // gated: [mtiles, R] chunks
  __nv_bfloat16 *gate, *up;       // gated, optional [T, R*B]
  const float* dh;                // backward: [T, R*B]
  __nv_bfloat16* dgu;             // backward: [T, 2*R*B], d_gate then d_up
  void* out;                      // linear [T, R*B]
  const void* residual;           // linear, optional, out's type
  int32_t out_f32;
  int32_t wide;                   // out, residual, gate and up are 32-byte aligned
  int32_t split;                  // linear: CTAs sharing a unit (0: persistent, whole units)
  int32_t early;                  // weights, plan and residual were complete before the kernel ahead
  int32_t* status;
  uint64_t timeout_ns;
};

struct Smem {
  uint8_t* stages;
  uint64_t *full, *empty, *acc_full, *acc_empty, *drain;
  uint32_t *count, *tmem_slot;  // live slots of each stage
  volatile int* abort_flag;
};

template <class G>
__device__ __forceinline__ Smem carve(uint8_t* raw) {
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

// The CTA's units are blockIdx.x + i * gridDim.x, a unit being a block-row of a
// token tile (kPairs: of two).  Issuer k's job i is unit i of matrix k (gated),
// of tile k of the two, or unit 2i + k (linear).  In split mode a ring has one
// job, stages [first, first + stages) of the cluster's unit.
struct RingWork {
  int jobs, first, stages;
};
template <class G>
__device__ __forceinline__ int all_units(const Params& p) {
  return (p.mtiles + G::TILES - 1) / G::TILES * p.R;
}
template <class G>
__device__ __forceinline__ RingWork ring_work(const Params& p, int k) {
  const int K = G::GATED && k ? p.K1 : p.K0;
  const int all = (K + G::SLOTS - 1) / G::SLOTS;
  if (!G::GATED && p.split) {
    const int part = int(blockIdx.x) % p.split * 2 + k, each = (all + 2 * p.split - 1) / (2 * p.split);
    return {1, part * each, max(0, min(each, all - part * each))};
  }
  const int units = all_units<G>(p), grid = int(gridDim.x);
  const int mine = int(blockIdx.x) < units ? (units - int(blockIdx.x) + grid - 1) / grid : 0;
  return {G::GATED || G::PAIRS ? mine : (mine - k + 1) / 2, 0, all};
}
template <class G>
__device__ __forceinline__ int job_unit(const Params& p, int i, int k) {
  if (!G::GATED && p.split) return int(blockIdx.x) / p.split;
  return int(blockIdx.x) + (G::GATED || G::PAIRS ? i : 2 * i + k) * int(gridDim.x);
}

// ------------------------------------------------------------- direct rows
//
// Few rows come as they are (no chunks in memory, and no launch to write them):
// each CTA quantises the columns that its slots take, into the stages.  The
// epilogue's warps, idle until the first accumulator, do so for the rings'
// first filling, all slots and row groups at once; the producers for the uses
// after it.

// Rows [n0, n0 + N), N = 8 or 16, of the chunk of column block c: a lane takes a
// scale block of a row, as in the quantisation kernel.
template <int B>
struct DirectRows {
  static constexpr int N = 32 * kBlock / B;
  static __device__ __forceinline__ void put(const Params& p, int c, int n0, uint8_t* chunk) {
    const int lane = threadIdx.x & 31;
    const int j = (lane >> 3) & (B / kBlock - 1), n = n0 + (lane & 7) + (B == 64 ? (lane >> 4) * 8 : 0);
    if (n >= int(p.T)) return;
    float v[32];
    const int64_t at = n * p.ld_src + int64_t(c) * B + j * kBlock;
    if (p.src_f32)
      load32(static_cast<const float*>(p.src) + at, v);
    else
      load32(static_cast<const __nv_bfloat16*>(p.src) + at, v);
    uint32_t byte;
    *reinterpret_cast<uint4*>(chunk + code_off(n, j, kRows * 32)) = quantize32(v, byte);
    chunk[kRows * B / 2 + scale_off(n, j)] = uint8_t(byte);
  }
};

// The epilogue warps and the producers, once, after the first filling's rows.
__device__ __forceinline__ void direct_barrier() {
  asm volatile("bar.sync 1, %0;" ::"n"(32 * (kProducers + kEpiWarps)) : "memory");
}

template <int B, class G>
__device__ void direct_first(const Params& p, const Smem& s) {
  const int w = (threadIdx.x >> 5) - kProducers;
  const int groups = (int(p.T) + DirectRows<B>::N - 1) / DirectRows<B>::N;
  for (int item = w; item < G::NS * G::SLOTS * groups; item += kEpiWarps) {
    const int n0 = item % groups * DirectRows<B>::N, at = item / groups;
    const int i = at % G::SLOTS, use = at / G::SLOTS % G::NR, ring = at / (G::SLOTS * G::NR);
    const RingWork rw = ring_work<G>(p, ring);
    const int job = rw.stages > 0 ? use / rw.stages : rw.jobs;
    if (job >= rw.jobs) continue;
    const int u = job_unit<G>(p, job, ring), r = u % p.R;
    const int mat = G::GATED ? ring : 0, K = mat ? p.K1 : p.K0, k = (rw.first + use - job * rw.stages) * G::SLOTS + i;
    const uint32_t e = k < K ? __ldg((mat ? p.p1 : p.p0).entries + int64_t(r) * K + k) : kNoSlot;
    if (e != kNoSlot) DirectRows<B>::put(p, int(e & 0xFFFFu), n0, s.stages + (ring * G::NR + use) * G::STAGE + i * G::SLOT);
  }
  fence_proxy_async_smem();
  direct_barrier();
}

// ---------------------------------------------------------------- producer

template <int B, class G>
__device__ void produce(const Params& p, const Smem& s, int ring, int sub, const Ctl& ctl) {
  const int lane = threadIdx.x & 31;
  const uint64_t keep = policy_evict_last(), pass = policy_evict_normal();
  const int mat = G::GATED ? ring : 0;
  const int K = mat ? p.K1 : p.K0;
  const uint8_t* w = mat ? p.w1 : p.w0;
  const uint32_t* entries = (mat ? p.p1 : p.p0).entries;
  const RingWork rw = ring_work<G>(p, ring);
  uint64_t* full = s.full + ring * G::NR;
  uint64_t* empty = s.empty + ring * G::NR;
  uint32_t* count = s.count + ring * G::NR;
  uint8_t* stages = s.stages + ring * (G::NR * G::STAGE);
  int job = 0, part = sub, left = rw.stages > 0 ? rw.jobs : 0;  // of the next use
  while (part >= rw.stages && job < left) {
    part -= rw.stages;
    ++job;
  }
  // Two lanes (kPairs: three) bring a slot of a stage, its rows and its weights:
  // one copy instruction for all of a stage's copies.  (One lane after another's
  // took 700 cycles a stage, which the stages spend empty.)
  constexpr int LANES = G::TILES + 1;
  const int slot = lane / LANES, piece = lane - slot * LANES;
  const bool is_w = piece == G::TILES;
  struct Use {
    uint32_t e;           // this lane's slot's entry
    const uint8_t* base;  // of its chunks
  };
  // units advance by a fixed step: block-row and token tile without divisions
  const int step = job_unit<G>(p, 1, ring) - job_unit<G>(p, 0, ring), dm = step / p.R, dr = step - dm * p.R;
  int m = job_unit<G>(p, job, ring) / p.R, r = job_unit<G>(p, job, ring) - m * p.R;
  auto fetch = [&]() -> Use {
    const int k = (rw.first + part) * G::SLOTS + slot;
    const uint32_t e = lane < LANES * G::SLOTS && k < K ? __ldg(entries + int64_t(r) * K + k) : kNoSlot;
    // an odd last tile is its own neighbour (the epilogue stores it once)
    const int mt = G::PAIRS ? min(2 * m + piece, p.mtiles - 1) : m;
    return {e, is_w ? w + int64_t(r) * K * G::W : p.x + int64_t(mt) * p.C * G::A};
  };
  auto advance = [&] {
    part += G::PER;
    while (part >= rw.stages && job < left) {
      part -= rw.stages;
      ++job;
      m += dm;
      r += dr;
      if (r >= p.R) {
        r -= p.R;
        ++m;
      }
    }
  };
  auto copies = [&](const Use& use, uint32_t stage, bool weights, bool rows) {
    const bool live = use.e != kNoSlot;
    const uint32_t cnt = uint32_t(__popc(__ballot_sync(0xffffffffu, live))) / uint32_t(LANES);
    uint8_t* st = stages + stage * uint32_t(G::STAGE);
    uint8_t* to = st + slot * G::SLOT + piece * G::A;
    const uint8_t* from = use.base + (is_w ? int64_t(use.e >> 16) * G::W : int64_t(use.e & 0xFFFFu) * G::A);
    if (weights && elect_one()) {
      count[stage] = cnt;
      if (!p.x)
        mbar_expect_tx(&full[stage], cnt * uint32_t(G::W));
      else if (cnt)
        mbar_arrive_expect_tx(&full[stage], cnt * uint32_t(G::SLOT));
      else
        mbar_arrive(&full[stage]);
    }
    __syncwarp();
    if (live && (is_w ? weights : rows && p.x != nullptr))
      bulk_load(to, from, is_w ? G::W : G::A, &full[stage], is_w ? keep : pass);
    if (!p.x && rows) {  // direct rows, this warp's (with `rows` false they are already on their way)
      for (int i = 0; i < int(cnt); ++i) {
        const int c = int(__shfl_sync(0xffffffffu, use.e, LANES * i) & 0xFFFFu);
        for (int n0 = 0; n0 < int(p.T); n0 += DirectRows<B>::N) DirectRows<B>::put(p, c, n0, st + i * G::SLOT);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (elect_one()) mbar_arrive(&full[stage]);
    }
    __syncwarp();
  };
  uint32_t stage = uint32_t(sub), phase = 0;
  int64_t filled = 0;
  auto turn = [&] {
    ++filled;
    stage += G::PER;
    if (stage >= uint32_t(G::NR)) {
      stage -= G::NR;
      phase ^= 1u;
    }
  };
  // The ring's first filling: the weights need not wait for the rows, which the
  // kernel ahead or the epilogue's warps make.
  if (p.early || !p.x) {
    Use first[(G::NR + G::PER - 1) / G::PER];
    int n = 0;
#pragma unroll
    for (int i = 0; i < (G::NR + G::PER - 1) / G::PER; ++i) {
      if (sub + G::PER * i < G::NR && job < left) {
        first[i] = fetch();
        advance();
        copies(first[i], uint32_t(sub + G::PER * i), true, false);
        n = i + 1;
      }
    }
    if (p.x)
      griddep_wait();
    else
      direct_barrier();
#pragma unroll
    for (int i = 0; i < (G::NR + G::PER - 1) / G::PER; ++i) {
      if (i < n) {
        if (p.x)
          copies(first[i], uint32_t(sub + G::PER * i), false, true);
        else if (elect_one())
          mbar_arrive(&full[sub + G::PER * i]);
        turn();
      }
    }
    __syncwarp();
  }
  // from here each use's entries travel while the one before is issued
  Use next{kNoSlot, nullptr};
  if (job < left) next = fetch();
  bool ok = true;
  while (job < left) {
    const Use use = next;
    advance();
    if (job < left) next = fetch();
    ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1u, ctl));
    if (!ok) break;
    copies(use, stage, true, true);
    turn();
  }
  if (!ok && lane == 0) {  // let this producer's copies land before the CTA exits (bounded)
    for (int i = 0; i < G::NR && filled > 0; ++i, --filled) {
      if (stage < uint32_t(G::PER)) {
        stage += G::NR;
        phase ^= 1u;
      }
      stage -= G::PER;
      const uint32_t a = smem_u32(&full[stage]);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(a, phase) && globaltimer_ns() - t0 < 100000000ull) {
      }
    }
  }
}

// ------------------------------------------------------------------ issuer

template <int B, class G>
__device__ void issue(const Params& p, const Smem& s, uint32_t tmem, int k, const Ctl& ctl) {
  const bool leader = elect_one();
  const int ring = G::PAIRS ? 0 : k;
  constexpr uint32_t w_at = G::TILES * G::A;          // of a slot: its weights
  const uint32_t a_at = G::PAIRS ? uint32_t(k * G::A) : 0u;  // and this issuer's rows
  const uint32_t a0 = sdesc_lo(smem_u32(s.stages) + ring * (G::NR * G::STAGE), 128);
  const uint32_t sf0 = sdesc_lo(smem_u32(s.stages) + ring * (G::NR * G::STAGE), 16);
  const RingWork rw = ring_work<G>(p, k);
  uint64_t* full = s.full + ring * G::NR;
  uint64_t* empty = s.empty + ring * G::NR;
  uint32_t stage = 0, phase = 0;
  uint32_t acc = uint32_t(k), use = 0;  // job 2i + k of the CTA: accumulator (2i + k) % ACCS
  bool ok = true;
  for (int i = 0; i < rw.jobs && ok; ++i) {
    ok = __all_sync(0xffffffffu, mbar_wait(&s.acc_empty[acc], (use & 1u) ^ 1u, ctl));
    if (!ok) break;
    tc_fence_after();
    const uint32_t d = tmem + acc * B;
    uint32_t more = 0;
    for (int part = 0; part < rw.stages; ++part) {
      ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, ctl));
      if (!ok) break;
      tc_fence_after();
      const int n = int(s.count[ring * G::NR + stage]);
      if (leader) {
        const uint32_t st = stage * uint32_t(G::STAGE >> 4);
        const uint32_t sf = tmem + G::SF_COL + (uint32_t(k) * G::NR + stage) * G::SF_STAGE;
#pragma unroll
        for (int j = 0; j < G::SLOTS; ++j) {
          if (j < n) {
            const uint32_t at = st + j * (G::SLOT >> 4);
            copy_scales(sf + j * 8, sf0 + at + ((a_at + G::A - kScaleBytes) >> 4));
            copy_scales(sf + j * 8 + 4, sf0 + at + ((G::SLOT - kScaleBytes) >> 4));
#pragma unroll
            for (int kk = 0; kk < B / 64; ++kk)
              mma_mxf4(d, a0 + at + ((a_at + kk * kRows * 32) >> 4), a0 + at + ((w_at + kk * B * 32) >> 4),
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
    mma_commit(&s.drain[k]);
    const uint32_t a = smem_u32(&s.drain[k]);
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(a, 0) && globaltimer_ns() - t0 < 100000000ull) {
    }
  }
  __syncwarp();
}

// ---------------------------------------------------------------- epilogue

// silu(g) = g / (1 + e^-g) in fp32, two at a time.  Relative error at most
// 1.25 |g| 2^-24 + 2^-21: the exponent -g log2(e) is rounded once (and its
// constant), which e^-g magnifies by |g|; the exponential, the reciprocal, the
// sum and the product add the rest.  That is 1.6e-6 at g = -15 and 6e-6 at -80.
// The hardware tanh form of the bf16 kernels (2^-11) would move one in a few
// hundred of h's 4-bit codes to a neighbour.  Subnormal intermediates are
// flushed: e^-g below 2^-126 next to 1, and 1 / (1 + e^-g) below 2^-126, so that
// silu is zero for g below -87.3 (an absolute error below 2^-119).
__device__ __forceinline__ float2 silu2(float2 g) {
  const float2 t = mul2(g, make_float2(-1.4426950408889634f, -1.4426950408889634f));
  float2 e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
  const float2 a = add2(e, make_float2(1.f, 1.f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(a.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(a.y));
  return mul2(g, r);
}

// This warp has read accumulator `acc`.
__device__ __forceinline__ void release(const Smem& s, uint32_t acc) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(&s.acc_empty[acc]);
}

// A projection without a live slot is zero.
__device__ __forceinline__ void clear16(uint32_t (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = 0u;
}

__device__ __forceinline__ void put_bf16(__nv_bfloat16* o, const uint32_t (&v)[16], bool wide) {
  uint32_t a[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) a[e] = pack_bf16x2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]));
  if (wide) {
    st_global_v8(o, a);
  } else {
    st_global_v4(o, a[0], a[1], a[2], a[3]);
    st_global_v4(o + 8, a[4], a[5], a[6], a[7]);
  }
}

// Sixteen outputs of a linear at element `at`: the residual, one rounding, the
// stores.  A lane's outputs lie 2 or 4 KB and more from the next lane's, so its
// accesses fill sectors only if they are 32 bytes (p.wide: the buffers are
// aligned so; else two of 16).
__device__ __forceinline__ void put8(const Params& p, int64_t at, float* f) {  // fp32: 8 values are 32 bytes
  uint32_t r[8];
  if (p.residual) {
    const float* from = static_cast<const float*>(p.residual) + at;
    if (p.wide) {
      ld_global_v8(from, r);
    } else {
      const uint4 a = ld_global_v4(from), b = ld_global_v4(from + 4);
      r[0] = a.x, r[1] = a.y, r[2] = a.z, r[3] = a.w, r[4] = b.x, r[5] = b.y, r[6] = b.z, r[7] = b.w;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] += __uint_as_float(r[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(f[i]);
  float* o = static_cast<float*>(p.out) + at;
  if (p.wide) {
    st_global_v8(o, r);
  } else {
    st_global_v4(o, r[0], r[1], r[2], r[3]);
    st_global_v4(o + 4, r[4], r[5], r[6], r[7]);
  }
}
__device__ __forceinline__ void put16(const Params& p, int64_t at, float* f) {
  if (p.out_f32) {
    put8(p, at, f);
    put8(p, at + 8, f + 8);
    return;
  }
  uint32_t r[8];
  if (p.residual) {
    const __nv_bfloat16* from = static_cast<const __nv_bfloat16*>(p.residual) + at;
    if (p.wide) {
      ld_global_v8(from, r);
    } else {
      const uint4 a = ld_global_v4(from), b = ld_global_v4(from + 8);
      r[0] = a.x, r[1] = a.y, r[2] = a.z, r[3] = a.w, r[4] = b.x, r[5] = b.y, r[6] = b.z, r[7] = b.w;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 x = unpack_bf16x2(r[i]);
      f[2 * i] += x.x;
      f[2 * i + 1] += x.y;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + at;
  if (p.wide) {
    st_global_v8(o, r);
  } else {
    st_global_v4(o, r[0], r[1], r[2], r[3]);
    st_global_v4(o + 8, r[4], r[5], r[6], r[7]);
  }
}

// Split mode.  Each CTA leaves the sum of its two accumulators in the ring's
// shared memory (free: every copy into it has been consumed), rows of B + 4
// floats; then CTA `rank` of the cluster adds columns [rank * B / split, ...)
// of all of them, in rank order.
template <int B>
struct Partial {
  static constexpr int LD = B + 4;
  static_assert(kRows * LD * 4 <= Geo<B, kLinear>::NS * Geo<B, kLinear>::STAGE, "the partial sums fit the ring");
};

template <int B>
__device__ void split_partial(const Params& p, const Smem& s, uint32_t tmem, const Ctl& ctl) {
  using G = Geo<B, kLinear>;
  const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) - kProducers;
  const int q = int(threadIdx.x >> 5) & 3, j = w >> 2;
  if (j >= B / 32) return;  // one unit: the second group of B = 64 has none
  const int u = int(blockIdx.x) / p.split, m = u / p.R, r = u - m * p.R;
  const int n = q * 32 + lane;
  const int live = __ldg(p.p0.counts + r);
  float f[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) f[i] = 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (!__all_sync(0xffffffffu, mbar_wait(&s.acc_full[k], 0, ctl))) return;
    tc_fence_after();
    uint32_t a[32];
    tmem_ld32_sync(tmem + (uint32_t(q * 32) << 16) + uint32_t(k * B + j * 32), a);
    const RingWork rw = ring_work<G>(p, k);
    if (rw.stages > 0 && live > rw.first * G::SLOTS) {
#pragma unroll
      for (int i = 0; i < 32; ++i) f[i] += __uint_as_float(a[i]);
    }
  }
  if (int64_t(m) * kRows + n >= p.T) return;
  float* row = reinterpret_cast<float*>(s.stages) + n * Partial<B>::LD + j * 32;
#pragma unroll
  for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(row + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
}

// Four outputs of a linear at element `at`.
__device__ __forceinline__ void put4(const Params& p, int64_t at, float4 f) {
  if (p.out_f32) {
    if (p.residual) {
      const float4 r = *reinterpret_cast<const float4*>(static_cast<const float*>(p.residual) + at);
      f.x += r.x, f.y += r.y, f.z += r.z, f.w += r.w;
    }
    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = f;
    return;
  }
  if (p.residual) {
    const uint2 r = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.residual) + at);
    const float2 a = unpack_bf16x2(r.x), b = unpack_bf16x2(r.y);
    f.x += a.x, f.y += a.y, f.z += b.x, f.w += b.y;
  }
  *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) =
      make_uint2(pack_bf16x2(f.x, f.y), pack_bf16x2(f.z, f.w));
}

// A thread joins four columns of a row: the loads of all ranks first, then the
// sum in rank order.
template <int B>
__device__ void split_join(const Params& p, const Smem& s) {
  const int u = int(blockIdx.x) / p.split, rank = int(blockIdx.x) % p.split, m = u / p.R, r = u - m * p.R;
  const int rows = int(min(int64_t(kRows), p.T - int64_t(m) * kRows));
  const int cols = B / p.split, per_row = cols / 4;
  const uint32_t base = smem_u32(s.stages);
  for (int i = threadIdx.x; i < rows * per_row; i += kThreads) {
    const int n = i / per_row, c = rank * cols + (i - n * per_row) * 4;
    float4 v[kMaxSplit];
#pragma unroll
    for (int k = 0; k < kMaxSplit; ++k) {
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k < p.split)
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[k].x), "=f"(v[k].y), "=f"(v[k].z), "=f"(v[k].w)
                     : "r"(mapa_shared(base + uint32_t(n * Partial<B>::LD + c) * 4u, uint32_t(k)))
                     : "memory");
    }
    float4 f = v[0];
#pragma unroll
    for (int k = 1; k < kMaxSplit; ++k) f.x += v[k].x, f.y += v[k].y, f.z += v[k].z, f.w += v[k].w;
    put4(p, (int64_t(m) * kRows + n) * (int64_t(p.R) * B) + int64_t(r) * B + c, f);
  }
}

// d_gate = d_h u silu'(g) and d_up = d_h silu(g), two at a time, fp32:
// silu' = s + silu (1 - s), s = 1 / (1 + e^-g).  They leave in bf16: they are
// operands of bf16 products (dx and two tile gradients, half of a step's time),
// and keeping them whole would take a second product of their low parts.  With
// the result's own rounding a tile gradient's error is 2.3e-3 instead of 1.65e-3.
__device__ __forceinline__ void silu_backward2(float2 dh, float2 g, float2 u, float2& dg, float2& du) {
  const float2 t = mul2(g, make_float2(-1.4426950408889634f, -1.4426950408889634f));
  float2 e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
  const float2 a = add2(e, make_float2(1.f, 1.f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(a.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(a.y));
  const float2 f = mul2(g, r);
  const float2 slope = add2(r, mul2(f, make_float2(1.f - r.x, 1.f - r.y)));
  dg = mul2(mul2(dh, u), slope);
  du = mul2(dh, f);
}

template <int B, Mode MODE>
__device__ void epilogue(const Params& p, const Smem& s, uint32_t tmem, const Ctl& ctl) {
  using G = Geo<B, MODE>;
  constexpr bool GATED = G::GATED;
  constexpr int NB = B / 32;             // scale blocks (32 features) of a unit
  constexpr int GROUPS = kEpiWarps / (4 * NB);
  constexpr int JOBS = GATED ? 2 : 1;
  const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) - kProducers;
  const int q = int(threadIdx.x >> 5) & 3, j = (w >> 2) % NB, group = (w >> 2) / NB;
  const int units = all_units<G>(p);
  const int64_t ld = int64_t(p.R) * B;
  const uint32_t lanes = uint32_t(q * 32) << 16;
  const int step = GROUPS * int(gridDim.x);
  uint32_t acc = uint32_t(group * JOBS * G::TILES), use = 0;  // accumulator of this unit's first job
  int c0 = 0, c1 = 0;  // live slots of the next unit's rows, read a unit ahead
  auto counts = [&](int r) {
    c0 = __ldg(p.p0.counts + r);
    if (GATED) c1 = __ldg(p.p1.counts + r);
  };
  auto next = [&](int jobs) {
    acc += jobs;
    while (acc >= uint32_t(G::ACCS)) {
      acc -= G::ACCS;
      ++use;
    }
  };
  int u = int(blockIdx.x) + group * int(gridDim.x);
  // the next unit's token tile and block-row, advanced without divisions
  const int dm = step / p.R, dr = step - dm * p.R;
  int mn = u / p.R, rn = u - mn * p.R;
  if (u < units) counts(rn);
  for (; u < units; u += step) {
    const int m = mn * G::TILES, r = rn;
    const int n = q * 32 + lane;
    const int64_t t = int64_t(m) * kRows + n;
    const bool live0 = c0 > 0, live1 = c1 > 0;
    mn += dm;
    rn += dr;
    if (rn >= p.R) {
      rn -= p.R;
      ++mn;
    }
    const bool more = u + step < units;
    if (more) counts(rn);
    const int64_t at = t * ld + int64_t(r) * B + j * 32;
    if constexpr (MODE == kGatedBackward) {
      const uint32_t a0 = acc, a1 = acc + 1 == uint32_t(G::ACCS) ? 0u : acc + 1;
      const uint32_t use1 = a1 ? use : use + 1;
      const uint32_t col = tmem + lanes + uint32_t(j * 32);
      const bool row = t < p.T;
      uint32_t dh[2][8] = {};  // 16 columns of d_h, on their way while the products run
      auto fetch = [&](int k) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (row) ld_global_v8(p.dh + at + k + 8 * i, dh[i]);
      };
      // a lane's 32 columns are one line of d_h: the next unit's is called into L2
      // now (this kernel waits for memory, not for its rate; without it 405 us
      // at T = 8192, d = 4096, d_ff = 16384)
      const int64_t tn = int64_t(mn) * kRows + n;
      if (more && tn < p.T)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p.dh + tn * ld + int64_t(rn) * B + j * 32));
      fetch(0);
      if (!__all_sync(0xffffffffu, mbar_wait(&s.acc_full[a0], use & 1u, ctl))) return;
      if (!__all_sync(0xffffffffu, mbar_wait(&s.acc_full[a1], use1 & 1u, ctl))) return;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < 32; k += 16) {
        uint32_t g[16], u[16];
        tmem_ld16x2_sync(col + a0 * B + k, g, col + a1 * B + k, u);
        if (k) {
          release(s, a0);
          release(s, a1);
        }
        if (!live0) clear16(g);
        if (!live1) clear16(u);
        uint32_t og[8], ou[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t* d = dh[i >> 2] + 2 * (i & 3);
          float2 x, y;
          silu_backward2(make_float2(__uint_as_float(d[0]), __uint_as_float(d[1])),
                         make_float2(__uint_as_float(g[2 * i]), __uint_as_float(g[2 * i + 1])),
                         make_float2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1])), x, y);
          og[i] = pack_bf16x2(x.x, x.y);
          ou[i] = pack_bf16x2(y.x, y.y);
        }
        if (!k) fetch(16);
        if (row) {
          __nv_bfloat16* o = p.dgu + t * 2 * ld + int64_t(r) * B + j * 32 + k;
          st_global_v8(o, og);
          st_global_v8(o + ld, ou);
        }
      }
    } else if constexpr (MODE == kGated) {
      const uint32_t a0 = acc, a1 = acc + 1 == uint32_t(G::ACCS) ? 0u : acc + 1;
      const uint32_t use1 = a1 ? use : use + 1;
      const uint32_t col = tmem + lanes + uint32_t(j * 32);
      float h[32];
      auto gates = [&](int k, uint32_t (&v)[16]) {  // h[k..k+16) = silu of the gate's columns
        if (!live0) clear16(v);
        if (p.gate && t < p.T) put_bf16(p.gate + at + k, v, p.wide);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float2 x = silu2(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
          h[k + i] = x.x;
          h[k + i + 1] = x.y;
        }
      };
      auto ups = [&](int k, uint32_t (&v)[16]) {  // times the up columns
        if (!live1) clear16(v);
        if (p.gate && t < p.T) put_bf16(p.up + at + k, v, p.wide);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float2 x = mul2(make_float2(h[k + i], h[k + i + 1]),
                                make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
          h[k + i] = x.x;
          h[k + i + 1] = x.y;
        }
      };
      // 16 columns at a time: 32 spill.  B = 128: the gate half is freed as soon
      // as it is read, so that the next unit's jobs wait less for one of the
      // three accumulators (gate/up at T = 16384, d = 4096, d_ff = 16384: 307 us
      // against 345 with both halves read together).  B = 64, two units in turn
      // on the epilogue's two groups, is bound by the epilogue and gains from
      // fewer waits (125 us together, 138 one after the other; d = 2048,
      // d_ff = 8192).
      if (!__all_sync(0xffffffffu, mbar_wait(&s.acc_full[a0], use & 1u, ctl))) return;
      if constexpr (B == 128) {
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 32; k += 16) {
          uint32_t v[16];
          tmem_ld16_sync(col + a0 * B + k, v);
          if (k) release(s, a0);
          gates(k, v);
        }
        if (!__all_sync(0xffffffffu, mbar_wait(&s.acc_full[a1], use1 & 1u, ctl))) return;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 32; k += 16) {
          uint32_t v[16];
          tmem_ld16_sync(col + a1 * B + k, v);
          if (k) release(s, a1);
          ups(k, v);
        }
      } else {
        if (!__all_sync(0xffffffffu, mbar_wait(&s.acc_full[a1], use1 & 1u, ctl))) return;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 32; k += 16) {
          uint32_t v[16], w[16];
          tmem_ld16x2_sync(col + a0 * B + k, v, col + a1 * B + k, w);
          if (k) {
            release(s, a0);
            release(s, a1);
          }
          gates(k, v);
          ups(k, w);
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
      for (int k = 0; k < G::TILES; ++k) {
        if (k) next(1);
        if (!__all_sync(0xffffffffu, mbar_wait(&s.acc_full[acc], use & 1u, ctl))) return;
        tc_fence_after();
        uint32_t a[32];
        tmem_ld32_sync(tmem + lanes + acc * B + j * 32, a);
        release(s, acc);
        if (t + k * kRows < p.T) {
          float f[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = live0 ? __uint_as_float(a[i]) : 0.f;
          put16(p, at + k * kRows * ld, f);
          put16(p, at + k * kRows * ld + 16, f + 16);
        }
      }
    }
    next(GROUPS * JOBS * G::TILES - (G::TILES - 1));  // this group's next unit
  }
}

template <int B, Mode MODE>
__global__ void __launch_bounds__(kThreads, 1) bell_mx_kernel(const Params p) {
  using G = Geo<B, MODE>;
  extern __shared__ uint8_t smem_raw[];
  const Smem s = carve<G>(smem_raw);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < G::NS; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 2 / G::RINGS);  // the issuers that take from it
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
  // Rows, and possibly weights, come from the kernel ahead.  With p.early only
  // the rows do, and the producers start the weights before they wait.  A kernel
  // on the caller's rows lets the next one start only when all before it is
  // complete: the next one's p.early rests on that.
  if (p.x) griddep_launch();
  if (!p.early || warp >= kProducers) griddep_wait();
  if (!p.x) griddep_launch();
  const bool split = MODE == kLinear && p.split;
  if (warp < kProducers) {
    if (warp < G::RINGS * G::PER) produce<B, G>(p, s, warp / G::PER, warp % G::PER, ctl);
  } else if (warp < kIssuer) {
    if constexpr (!G::PAIRS) {
      if (!p.x) direct_first<B, G>(p, s);
    }
    if constexpr (MODE == kLinear) {
      if (split) split_partial<B>(p, s, tmem, ctl);
    }
    if (!split) epilogue<B, MODE>(p, s, tmem, ctl);
  } else {
    issue<B, G>(p, s, tmem, warp - kIssuer, ctl);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (MODE == kLinear) {
    if (split) {
      cluster_sync();  // every partial sum is in place
      split_join<B>(p, s);
      cluster_sync();  // and has been read before its CTA leaves
    }
  }
  if (warp == kIssuer) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Slots of a row from which CTAs share a unit of a linear.  The cluster's launch
// and the join cost 2 us, more with more rows to join; a slot takes a whole unit
// 0.15 to 0.3 us, and 0.25 to 0.5 where it quantises its rows itself, which the
// mxfp4.py calls have it do up to 8 tokens at B = 128 and 32 at B = 64.  us whole
// and split (graph replays, quantisation included where it is a launch of its own):
//   B = 128, R = 32   T = 1: K = 16 7.5, 6.9; 32 12.0, 7.4; R = 16, K = 12 6.1, 6.6
//     T = 16: K = 24 8.7, 9.1; 28 9.2, 9.2; 32 9.9, 9.4   T = 32: 32 10.0, 10.2; 40 11.2, 10.9
//     T = 64: K = 36 10.8, 11.2; 44 12.1, 11.5   T = 128: K = 40 12.4, 13.5; 48 13.6, 13.7; 64 16.1, 14.1
//   B = 64, R = 16    T = 1: K = 16 5.2, 6.7; 24 7.3, 7.4; 32 9.3, 6.8   T = 32: K = 16 7.9, 8.9; 24 12.2, 10.4
//     T = 33: K = 40 8.5, 8.8; 64 10.3, 8.8   T = 128: K = 48 9.6, 10.4; 64 10.7, 10.7; 96 13.6, 11.3
static int split_from(int64_t T, int B) {
  if (T <= (B == 64 ? BELL_MX_DIRECT_ROWS : 8)) return B == 64 ? 24 : 16;
  return B == 64 ? 64 : 32 + int(std::min<int64_t>(std::max<int64_t>(T - 32, 0), 96) / 4);
}

// CTAs that share a unit: a power of two, 16 columns each to join, a stage for
// every ring, and all clusters at once (of 16 clusters of eight some wait for the
// others: B = 128, R = 16, K = 32, T = 1: 12.4 us with eight CTAs, 11.9 whole, 7.3
// with four).  fit[i]: clusters of 2 << i CTAs that run together.
static int split_of(int64_t units, int64_t T, int K, int stages, int sms, int B, const int (&fit)[3]) {
  if (units * 2 > sms || K < split_from(T, B)) return 0;
  int split = 1;
  for (int i = 0; i < 3; ++i)
    if (2 * split <= B / 16 && units * split * 2 <= sms && split * 4 <= stages && units <= fit[i]) split *= 2;
    else break;
  return split > 1 ? split : 0;
}

// Clusters of 2, 4 and 8 CTAs of `kern` that run at once on the current device.
static int clusters_at_once(const void* kern, int threads, int smem, int (&fit)[3]) {
  for (int i = 0; i < 3; ++i) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = unsigned(2 << i);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(unsigned(2 << i));
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = size_t(smem);
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&fit[i], kern, &cfg) != cudaSuccess) {
      (void)cudaGetLastError();
      return fail(BELL_ERR_LAUNCH, "cudaOccupancyMaxActiveClusters");
    }
  }
  return BELL_OK;
}

template <int B, Mode MODE>
static int launch(Params p, int32_t max_ctas, cudaStream_t s) {
  using G = Geo<B, MODE>;
  auto kern = bell_mx_kernel<B, MODE>;
  static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit has been raised
  static std::atomic<int> fits[64][3];    // and there, clusters at once
  int dev = 0, sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(BELL_ERR_LAUNCH, "cudaGetDevice");
  if (!(ready.load() >> dev & 1)) {
    if (int rc = set_smem(reinterpret_cast<const void*>(kern), G::SMEM)) return rc;
    if (MODE == kLinear) {
      int fit[3];
      if (int rc = clusters_at_once(reinterpret_cast<const void*>(kern), kThreads, G::SMEM, fit)) return rc;
      for (int i = 0; i < 3; ++i) fits[dev][i] = fit[i];
    }
    ready.fetch_or(uint64_t(1) << dev);
  }
  if (max_ctas > 0 && sms > max_ctas) sms = max_ctas;
  const int64_t units = (int64_t(p.mtiles) + G::TILES - 1) / G::TILES * p.R;
  const int fit[3] = {fits[dev][0], fits[dev][1], fits[dev][2]};
  p.split = MODE != kLinear ? 0 : split_of(units, p.T, p.K0, (p.K0 + G::SLOTS - 1) / G::SLOTS, sms, B, fit);
  const int64_t grid = p.split ? units * p.split : std::min<int64_t>(units, sms);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = G::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(p.split);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.split ? 2 : 1;
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

// Quantise the caller's rows first where it gave any and wants them in x.
template <class D>
static int quantize_source(const D* d, const BellMxEll& w, Params* p, void* stream) {
  if (!d->x_src) return BELL_OK;
  if (d->x) return bell_mx_quantize_rows(d->T, w.C * w.B, w.B, d->src_dtype, d->x_src, d->ld_src, d->x, stream);
  p->src = d->x_src;
  p->ld_src = d->ld_src;
  p->src_f32 = d->src_dtype == BELL_DTYPE_F32;
  return check_rows(d->T, w.C * w.B, w.B, d->src_dtype, d->x_src, d->x_src, d->ld_src);
}

template <class D>
static int check_source(const D* d) {
  if (d->T > 0 && !d->x && !(d->x_src && d->T <= BELL_MX_DIRECT_ROWS))
    return fail(BELL_ERR_ARG, "x may be NULL only with x_src and T <= BELL_MX_DIRECT_ROWS");
  return BELL_OK;
}

static int linear(Params p, const BellMxEll& w, const void* residual, void* out, int32_t out_dtype, int32_t max_ctas,
                  cudaStream_t s) {
  p.out = out;
  p.residual = residual;
  p.out_f32 = out_dtype == BELL_DTYPE_F32;
  p.wide = ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(residual)) & 31u) == 0;
  // Two token tiles to a unit where that leaves a unit for three of four SMs.
  // 16384 -> 4096, K = 32, us with one tile and with two: 160 units (80 pairs)
  // 12.5, 13.4; 256: 15.2, 13.4; 320: 19.8, 19.8; 512: 24.8, 21.3; 1024: 40, 36;
  // 4096: 148, 133.  B = 64, 2048 -> 8192, K = 4: 1024 units 9.8, 9.6; 2048: 14.6,
  // 13.2; 4224: 25.7, 22.1; 16384: 84, 72.  A tile alone (128 units, B = 128, K = 8)
  // 6.1, 7.3; three of them 9.9, 9.9; five 13.7, 13.5.
  int sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  if (max_ctas > 0 && sms > max_ctas) sms = max_ctas;
  const bool pairs = p.x && p.mtiles > 1 && int64_t(p.mtiles + 1) / 2 * p.R * 4 >= int64_t(sms) * 3;
  if (w.B == 64) return pairs ? launch<64, kPairs>(p, max_ctas, s) : launch<64, kLinear>(p, max_ctas, s);
  return pairs ? launch<128, kPairs>(p, max_ctas, s) : launch<128, kLinear>(p, max_ctas, s);
}

int gated_backward(int64_t T, const void* x, const BellMxEll& gate, const BellMxEll& up, const float* dh, void* dgu,
                   int32_t* status, cudaStream_t s) {
  if (int rc = check_ell(gate, "gate")) return rc;
  if (int rc = check_ell(up, "up")) return rc;
  if (int rc = check_size(T, gate.R)) return rc;
  if (!status) status = default_status_ptr();
  if (!status) return BELL_ERR_LAUNCH;
  Params p = base_params(T, gate, &up, x, status);
  p.dh = dh;
  p.dgu = static_cast<__nv_bfloat16*>(dgu);
  return gate.B == 128 ? launch<128, kGatedBackward>(p, 0, s) : launch<64, kGatedBackward>(p, 0, s);
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
  if (int rc = mx::check_source(d)) return rc;
  if (d->T > 0 && !d->out) return fail(BELL_ERR_ARG, "out must be non-NULL");
  if (!aligned16(d->x) || !aligned16(d->out) || !aligned16(d->residual))
    return fail(BELL_ERR_ALIGN, "x, out and residual must be 16-byte aligned");
  if (d->max_ctas < 0) return fail(BELL_ERR_ARG, "max_ctas must be >= 0");
  if (int rc = require_sm100()) return rc;
  if (d->T == 0) return BELL_OK;
  int32_t* status = d->status ? d->status : default_status_ptr();
  if (!status) return BELL_ERR_LAUNCH;
  mx::Params p = mx::base_params(d->T, d->w, nullptr, d->x, status);
  if (int rc = mx::quantize_source(d, d->w, &p, stream)) return rc;
  // early: the quantisation ahead of the product is a plain launch, so all that
  // came before it is complete when the product starts
  p.early = d->x && d->x_src;
  return mx::linear(p, d->w, d->residual, d->out, d->out_dtype, d->max_ctas, static_cast<cudaStream_t>(stream));
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
  if (int rc = mx::check_source(d)) return rc;
  if (d->T > 0 && (!d->h || !d->out)) return fail(BELL_ERR_ARG, "h and out must be non-NULL");
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
  mx::Params p = mx::base_params(d->T, g, &u, d->x, status);
  if (int rc = mx::quantize_source(d, g, &p, stream)) return rc;
  p.h = static_cast<uint8_t*>(d->h);
  p.gate = static_cast<__nv_bfloat16*>(d->gate_pre);
  p.up = static_cast<__nv_bfloat16*>(d->up_out);
  p.wide = ((reinterpret_cast<uintptr_t>(d->gate_pre) | reinterpret_cast<uintptr_t>(d->up_out)) & 31u) == 0;
  p.early = d->x && d->x_src;
  if (int rc = g.B == 128 ? mx::launch<128, mx::kGated>(p, d->max_ctas, s) : mx::launch<64, mx::kGated>(p, d->max_ctas, s)) return rc;
  mx::Params q = mx::base_params(d->T, w, nullptr, d->h, status);
  // what came before the quantisation (a plain launch) or before gate/up on the
  // caller's rows is complete when the kernel ahead of this one lets it start
  q.early = d->x_src != nullptr;
  return mx::linear(q, w, d->residual, d->out, d->out_dtype, d->max_ctas, s);
}

}  // extern "C"
