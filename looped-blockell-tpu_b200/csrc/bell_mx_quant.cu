// bell_mx_quant.cu — MXFP4 quantisation and its inverse: activation rows,
// Block-ELL tiles and the plan of their live slots (layouts: bell_mx.cuh).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <string>

#include "bell_mx.cuh"

namespace bell {
namespace mx {

static constexpr int kThr = 256;

// Q(v) is a 2-bit significand times a power of two: exact in bf16 and fp32.

// Rows: a warp takes groups of 8 rows x 128 columns.
struct RowsArgs {
  int64_t T;
  int32_t features, C, B;
  int64_t groups;   // ceil(T / 8) * ceil(features / 128)
  int32_t col_groups;
};

// Group w's index without its columns, and the first column.
__device__ __forceinline__ int64_t split_off(const RowsArgs& a, int64_t w, int32_t& f0) {
  // a 64-bit division costs more than a group's other arithmetic
  const int64_t q = a.groups <= 0xFFFFFFFFll ? int64_t(uint32_t(w) / uint32_t(a.col_groups)) : w / a.col_groups;
  f0 = int32_t(w - q * a.col_groups) * 128;
  return q;
}

// Eight consecutive values, and the largest magnitude's fp32 bits (NaN on top).
// bf16 magnitudes compare as packed 16-bit integers.
struct Eight16 {
  uint4 w;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { w = ld_global_nc_v4(p); }
  __device__ __forceinline__ uint32_t top() const {
    const uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu), __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu));
    return max(m << 16, m & 0xFFFF0000u);
  }
  __device__ __forceinline__ float2 two(int i) const { return unpack_bf16x2(i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w); }
};
struct Eight32 {
  uint4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = ld_global_nc_v4(p);
    b = ld_global_nc_v4(p + 4);
  }
  __device__ __forceinline__ uint32_t top() const {
    const uint32_t m = 0x7FFFFFFFu;
    return max(max(max(a.x & m, a.y & m), max(a.z & m, a.w & m)), max(max(b.x & m, b.y & m), max(b.z & m, b.w & m)));
  }
  __device__ __forceinline__ float2 two(int i) const {
    return i == 0   ? make_float2(__uint_as_float(a.x), __uint_as_float(a.y))
           : i == 1 ? make_float2(__uint_as_float(a.z), __uint_as_float(a.w))
           : i == 2 ? make_float2(__uint_as_float(b.x), __uint_as_float(b.y))
                    : make_float2(__uint_as_float(b.z), __uint_as_float(b.w));
  }
};
template <class E>
struct EightOf;
template <>
struct EightOf<__nv_bfloat16> {
  using T = Eight16;
};
template <>
struct EightOf<float> {
  using T = Eight32;
};

// Quantise.  In pass p a lane takes eight values of row 2p + l / 16: a pass's
// loads are whole rows of 128 columns, and four lanes (word k = l % 4) share a
// scale block.  (One lane to a block, its loads 64 bytes apart from the next
// lane's, read fp32 at 4.6 TB/s instead of 6.4.)  The four lanes then exchange
// their words, so that lane k has all 16 bytes of pass k, and eight rows' stores
// fill a core matrix (128 bytes).  T = 8192, d = 16384: 67 us, 5.1 TB/s (T = 16384
// 126 us, 5.4 TB/s), where dequantisation, which computes little, reaches 5.5
// (5.7); the ALU is 74 % busy with 13 instructions a value, and without the
// maxima it took 65 us, so that memory is the nearer bound.
template <class E>
__global__ void __launch_bounds__(kThr) bell_mx_quantize_kernel(RowsArgs a, const E* __restrict__ src, int64_t ld,
                                                               uint8_t* __restrict__ dst) {
  griddep_launch();
  const int lane = threadIdx.x & 31, k = lane & 3, block = (lane >> 2) & 3, odd = lane >> 4;
  for (int64_t w = (int64_t(blockIdx.x) * kThr + threadIdx.x) >> 5; w < a.groups; w += int64_t(gridDim.x) * (kThr / 32)) {
    int32_t f0;
    const int64_t t0 = split_off(a, w, f0) * 8 + odd;
    const int32_t f = f0 + (lane & 15) * 8;
    const E* from = src + t0 * ld + f;
    typename EightOf<E>::T v[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      v[p] = {};
      if (t0 + 2 * p < a.T && f < a.features) v[p].load(from + 2 * p * ld);
    }
    uint32_t code[4], mine = 0;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      uint32_t top = v[p].top();
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t byte = scale_byte(top);
      if (p == k) mine = byte;
      const float inv = scale_inverse(byte);
      float s[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 t = mul2(v[p].two(i), make_float2(inv, inv));
        s[2 * i] = t.x;
        s[2 * i + 1] = t.y;
      }
      code[p] = pack_e2m1(s);
    }
    // 4 x 4 exchange: halves of two lanes, then single words
    const uint32_t x0 = __shfl_xor_sync(0xffffffffu, k & 2 ? code[0] : code[2], 2);
    const uint32_t x1 = __shfl_xor_sync(0xffffffffu, k & 2 ? code[1] : code[3], 2);
    // passes (k & 2) and (k & 2) + 1 of words k & ~2 and k | 2
    const uint32_t e0 = k & 2 ? x0 : code[0], e1 = k & 2 ? x1 : code[1];
    const uint32_t h0 = k & 2 ? code[2] : x0, h1 = k & 2 ? code[3] : x1;
    const uint32_t y0 = __shfl_xor_sync(0xffffffffu, k & 1 ? e0 : e1, 1);
    const uint32_t y1 = __shfl_xor_sync(0xffffffffu, k & 1 ? h0 : h1, 1);
    const uint4 q = k & 1 ? make_uint4(y0, e1, y1, h1) : make_uint4(e0, y0, h0, y1);
    // the scales of one row and column block are adjacent bytes: two (B = 64)
    // or four (B = 128) blocks' bytes leave as one store
    uint32_t word = mine | (__shfl_xor_sync(0xffffffffu, mine, 4) << 8);
    if (a.B == 128) word |= __shfl_xor_sync(0xffffffffu, word, 8) << 16;
    const int32_t fb = f0 + block * kBlock;
    const int64_t t = t0 + 2 * k;
    if (t < a.T && fb < a.features) {
      const int n = int(t & (kRows - 1)), c = fb / a.B, j = (fb - c * a.B) / kBlock;
      uint8_t* chunk = dst + (t / kRows * a.C + c) * row_chunk(a.B);
      st_global_v4(chunk + code_off(n, j, kRows * 32), q.x, q.y, q.z, q.w);
      if (j == 0) {
        uint8_t* p = chunk + a.B * (kRows / 2) + scale_off(n, 0);
        if (a.B == 128)
          *reinterpret_cast<uint32_t*>(p) = word;
        else
          *reinterpret_cast<uint16_t*>(p) = uint16_t(word);
      }
    }
  }
}

// Back: a lane's values fill one 16-byte store, and a warp's stores whole rows
// of 128 columns (256 or 512 contiguous bytes).
__device__ __forceinline__ void put_values(__nv_bfloat16* p, const uint8_t* codes, float s) {
  float v[8];
  unpack_e2m1(__ldg(reinterpret_cast<const unsigned*>(codes)), s, v);
  st_global_v4(p, pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void put_values(float* p, const uint8_t* codes, float s) {
  // four codes: half of an aligned word
  const uintptr_t at = reinterpret_cast<uintptr_t>(codes);
  const uint32_t w = __ldg(reinterpret_cast<const unsigned*>(at & ~uintptr_t(3))) >> ((at & 2u) * 8u);
  float v[8];
  unpack_e2m1(w, s, v);
  st_global_v4(p, __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}

template <class E>
__device__ __forceinline__ void dequantize_rows(const RowsArgs& a, const uint8_t* __restrict__ src, E* __restrict__ dst,
                                                int64_t ld) {
  constexpr int V = 16 / int(sizeof(E)), LANES = 128 / V, PASS = 32 / LANES;  // values a lane, lanes a row, rows a pass
  const int lane = threadIdx.x & 31;
  for (int64_t w = (int64_t(blockIdx.x) * kThr + threadIdx.x) >> 5; w < a.groups; w += int64_t(gridDim.x) * (kThr / 32)) {
    int32_t f0;
    const int64_t first = split_off(a, w, f0) * 8;
    const int32_t f = f0 + lane % LANES * V;
    if (f >= a.features) continue;
    const int c = f / a.B, j = (f - c * a.B) / kBlock, in = f % kBlock / 2;
    const uint8_t* chunk = src + (first / kRows * a.C + c) * row_chunk(a.B);
#pragma unroll
    for (int i = 0; i < 8; i += PASS) {
      const int64_t t = first + i + lane / LANES;
      const int n = int(t & (kRows - 1));
      if (t < a.T)
        put_values(dst + t * ld + f, chunk + code_off(n, j, kRows * 32) + in,
                   scale_value(chunk[a.B * (kRows / 2) + scale_off(n, j)]));
    }
  }
}

template <class E>
__global__ void __launch_bounds__(kThr) bell_mx_dequantize_kernel(RowsArgs a, const uint8_t* __restrict__ src,
                                                                 E* __restrict__ dst, int64_t ld) {
  dequantize_rows(a, src, dst, ld);
}

// One warp per block-row: the live slots, compacted in slot order.
__device__ __forceinline__ void plan_row(const int32_t* __restrict__ cols, int r, int32_t C, int32_t K,
                                         uint32_t* __restrict__ entries, int32_t* __restrict__ counts,
                                         int32_t* status) {
  const int lane = threadIdx.x & 31;
  int n = 0, bad = 0;
  for (int k0 = 0; k0 < K; k0 += 32) {
    const int k = k0 + lane;
    const int c = k < K ? cols[int64_t(r) * K + k] : -1;
    const bool live = c >= 0 && c < C;
    bad |= c < -1 || c >= C;
    const uint32_t m = __ballot_sync(0xffffffffu, live);
    if (live) entries[int64_t(r) * K + n + __popc(m & ((1u << lane) - 1u))] = uint32_t(c) | (uint32_t(k) << 16);
    n += __popc(m);
  }
  for (int k = n + lane; k < K; k += 32) entries[int64_t(r) * K + k] = kNoSlot;
  if (lane == 0) counts[r] = n;
  if (bad) atomicOr(status, BELL_STATUS_COLIDX);
}

struct PackWeight {
  const void* values;
  int64_t tiles;
  int32_t B, in_out;
  const int32_t* cols;
  int32_t R, C, K;
  uint8_t* chunks;
  uint32_t* entries;
  int32_t* counts;
  unsigned plan_end;  // blocks [.., plan_end) of the grid write the plan, a warp to a block-row
};
struct PackArgs {
  PackWeight w[BELL_MX_PACK_MAX];
  int32_t n;
  int32_t* status;
};

__device__ __forceinline__ void put_block(uint8_t* chunk, int B, int o, int j, const float (&v)[32]) {
  uint32_t byte;
  const uint4 q = quantize32(v, byte);
  st_global_v4(chunk + code_off(o, j, B * 32), q.x, q.y, q.z, q.w);
  chunk[B * B / 2 + scale_off(o, j)] = uint8_t(byte);
}

__device__ __forceinline__ float2 load_pair(const __nv_bfloat16* p) {
  return unpack_bf16x2(__ldg(reinterpret_cast<const unsigned*>(p)));
}
__device__ __forceinline__ float2 load_pair(const float* p) { return __ldg(reinterpret_cast<const float2*>(p)); }

// A thread takes the scale blocks j of two outputs of a tile.  [B_in, B_out]
// tiles are read a row of outputs at a time (lane = output pair): the 32 values
// of a block are strided and a warp's loads contiguous.
template <class E>
__global__ void __launch_bounds__(kThr) bell_mx_pack_kernel(const PackArgs a) {
  const unsigned plans = a.w[a.n - 1].plan_end;
  if (blockIdx.x < plans) {
    int i = 0;
    while (blockIdx.x >= a.w[i].plan_end) ++i;
    const PackWeight& w = a.w[i];
    const int r = int(blockIdx.x - (i ? a.w[i - 1].plan_end : 0u)) * (kThr / 32) + int(threadIdx.x >> 5);
    if (r < w.R) plan_row(w.cols, r, w.C, w.K, w.entries, w.counts, a.status);
    return;
  }
  for (int i = 0; i < a.n; ++i) {
    const PackWeight& p = a.w[i];
    const int B = p.B, blocks = B / kBlock, per_tile = B / 2 * blocks;
    const int64_t stride = int64_t(gridDim.x - plans) * kThr, n = p.tiles * per_tile;
    for (int64_t at = int64_t(blockIdx.x - plans) * kThr + threadIdx.x; at < n; at += stride) {
      const int64_t tile = at / per_tile;
      const int e = int(at - tile * per_tile);
      const E* v0 = static_cast<const E*>(p.values) + tile * B * B;
      uint8_t* ch = p.chunks + tile * tile_chunk(B);
      float v[32], w[32];
      if (p.in_out) {
        const int o = e % (B / 2) * 2, j = e / (B / 2);
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const float2 f = load_pair(v0 + (j * kBlock + k) * B + o);
          v[k] = f.x;
          w[k] = f.y;
        }
        put_block(ch, B, o, j, v);
        put_block(ch, B, o + 1, j, w);
      } else {
        const int j = e % blocks, o = e / blocks * 2;
        load32(v0 + o * B + j * kBlock, v);
        load32(v0 + (o + 1) * B + j * kBlock, w);
        put_block(ch, B, o, j, v);
        put_block(ch, B, o + 1, j, w);
      }
    }
  }
}

// Tiles back to bf16 [B_out, B_in], eight values a thread.
__device__ __forceinline__ void unpack_tiles(const TileGather& g, int32_t B) {
  const int per_row = B / 8, per_tile = B * per_row;
  __nv_bfloat16* values = static_cast<__nv_bfloat16*>(g.values);
  for (int64_t i = int64_t(blockIdx.x) * kThr + threadIdx.x; i < g.tiles * per_tile; i += int64_t(gridDim.x) * kThr) {
    const int64_t tile = i / per_tile;
    const int e = int(i - tile * per_tile), o = e / per_row, k = e % per_row * 8, j = k / kBlock;
    const int64_t from = g.index ? g.index[tile] : tile;
    if (from < 0 || from >= g.n0 + g.n1) continue;
    const uint8_t* ch = static_cast<const uint8_t*>(from < g.n0 ? g.c0 : g.c1) + (from < g.n0 ? from : from - g.n0) * tile_chunk(B);
    put_values(values + tile * B * B + o * B + k, ch + code_off(o, j, B * 32) + k % kBlock / 2,
               scale_value(ch[B * B / 2 + scale_off(o, j)]));
  }
}

__global__ void __launch_bounds__(kThr) bell_mx_unpack_kernel(const TileGather g, int32_t B) { unpack_tiles(g, B); }

// What a backward needs before its products, in one launch: gathered tiles and
// rows.
struct ExpandKernelArgs {
  ExpandArgs e;
  RowsArgs rows[2];
};
__global__ void __launch_bounds__(kThr) bell_mx_expand_kernel(const ExpandKernelArgs a) {
  for (int i = 0; i < 2; ++i)
    if (a.e.gather[i].tiles) unpack_tiles(a.e.gather[i], a.e.B);
  for (int i = 0; i < 2; ++i)
    if (a.e.rows[i].dst)
      dequantize_rows(a.rows[i], static_cast<const uint8_t*>(a.e.rows[i].src), static_cast<__nv_bfloat16*>(a.e.rows[i].dst),
                      a.e.rows[i].features);
}

// Up to three tile gradients: the parts of their units onto the sums in CTA
// order, zeros into dead slots, and all of it to bf16.  A block takes 2048 values,
// all of one tile, a thread eight; two parts are on their way at once.  I: the
// type of its divisions, 64-bit ones only where the numbers need them (they
// cost more than all the rest: 115 us against 69 at 50 million values).
static constexpr int kFinish = 8 * kThr;

struct Eight {
  uint4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = ld_global_v4(p);
    b = ld_global_v4(p + 4);
  }
  __device__ __forceinline__ void add_to(float (&v)[8]) const {
    v[0] += __uint_as_float(a.x), v[1] += __uint_as_float(a.y), v[2] += __uint_as_float(a.z), v[3] += __uint_as_float(a.w);
    v[4] += __uint_as_float(b.x), v[5] += __uint_as_float(b.y), v[6] += __uint_as_float(b.z), v[7] += __uint_as_float(b.w);
  }
};

struct FinishKernelArgs {
  FinishArgs f;
  int64_t end[3];  // of each gradient's items among all
};

template <class I>
__global__ void __launch_bounds__(kThr) bell_mx_finish_kernel(const FinishKernelArgs a) {
  for (int64_t all = blockIdx.x; all < a.end[2]; all += gridDim.x) {
    const int which = (all >= a.end[0]) + (all >= a.end[1]);
    const TileGrad& g = a.f.g[which];
    const int64_t item = which ? all - a.end[which - 1] : all;
    const int tile_size = g.B * g.B, shift = g.B == 128 ? 3 : 1;  // 8 or 2 items a tile
    const int64_t tile = item >> shift;
    const int at = (int(item & ((1 << shift) - 1)) * kThr + int(threadIdx.x)) * 8;
    float* sums = g.sums + tile * tile_size + at;
    const int c = __ldg(g.cols + tile);
    Eight own;
    own.load(sums);  // of a dead slot, anything
    const bool live = c >= 0 && c < g.C;
    int parts = 0;
    const float* part = nullptr;
    const int64_t ld = int64_t(g.cuts.slots) * tile_size;
    if (g.parts) {
      // the shares that start inside the tile's unit: steps * b / grid, rounded
      // down, in (first, first + chunks)
      const I r = I(tile) / I(g.K), k = I(tile) - r * I(g.K), kp = k / I(g.cuts.slots);
      const I first = (r * I(g.cuts.KP) + kp) * I(g.cuts.chunks), steps = I(g.cuts.steps), grid = I(g.cuts.grid);
      const I b = ((first + 1) * grid + steps - 1) / steps;
      parts = int(((first + I(g.cuts.chunks)) * grid + steps - 1) / steps - b);
      part = g.parts + int64_t(b) * ld + int64_t(k - kp * I(g.cuts.slots)) * tile_size + at;
    }
    if (!live) parts = 0;
    if (!g.rounded && live && !parts) continue;
    float v[8] = {};
    if (live) own.add_to(v);
    for (int i = 0; i < parts; i += 2, part += 2 * ld) {
      Eight w[2];
      w[0].load(part);
      if (i + 1 < parts) w[1].load(part + ld);
      w[0].add_to(v);
      if (i + 1 < parts) w[1].add_to(v);
    }
    if (g.rounded) {
      st_global_v4(static_cast<__nv_bfloat16*>(g.rounded) + tile * tile_size + at, pack_bf16x2(v[0], v[1]),
                   pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    } else {
      st_global_v4(sums, __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      st_global_v4(sums + 4, __float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
    }
  }
}

__global__ void __launch_bounds__(kThr) bell_mx_add_kernel(const float* a, const float* b, int64_t n, void* out, bool bf16) {
  for (int64_t i = (int64_t(blockIdx.x) * kThr + threadIdx.x) * 8; i < n; i += int64_t(gridDim.x) * kThr * 8) {
    Eight x, y;
    x.load(a + i);
    y.load(b + i);
    float v[8] = {};
    x.add_to(v);
    y.add_to(v);
    if (bf16) {
      st_global_v4(static_cast<__nv_bfloat16*>(out) + i, pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                   pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    } else {
      float* o = static_cast<float*>(out) + i;
      st_global_v4(o, __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      st_global_v4(o + 4, __float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
    }
  }
}

// Grid of grid-stride kernels: enough blocks for every SM's 2048 threads.
static int grid_for(int64_t threads, unsigned* grid) {
  int sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  const int64_t need = (threads + kThr - 1) / kThr, most = int64_t(sms) * 8 * 4;
  *grid = unsigned(need < most ? need : most);
  return BELL_OK;
}

int check_rows(int64_t T, int32_t features, int32_t B, int32_t dtype, const void* rows, const void* chunks,
                      int64_t ld) {
  if (B != 64 && B != 128) return fail(BELL_ERR_SHAPE, "MXFP4 rows: tile size B must be 64 or 128");
  if (T < 0 || T > (int64_t(1) << 31) - 256) return fail(BELL_ERR_SHAPE, "MXFP4 rows: T must be in [0, 2^31 - 256)");
  if (features < 1 || features % B) return fail(BELL_ERR_SHAPE, "MXFP4 rows: features must be a multiple of B");
  if (dtype != BELL_DTYPE_BF16 && dtype != BELL_DTYPE_F32) return fail(BELL_ERR_DTYPE, "MXFP4 rows: dtype must be bf16 or f32");
  if (T > 0 && (!rows || !chunks)) return fail(BELL_ERR_ARG, "MXFP4 rows: NULL buffer");
  if (ld < features || (ld * (dtype == BELL_DTYPE_BF16 ? 2 : 4)) % 16)
    return fail(BELL_ERR_ALIGN, "MXFP4 rows: the row stride must cover the features and be a multiple of 16 bytes");
  if (!aligned16(rows) || !aligned16(chunks)) return fail(BELL_ERR_ALIGN, "MXFP4 rows: buffers must be 16-byte aligned");
  return require_sm100();
}

static RowsArgs rows_args(int64_t T, int32_t features, int32_t B) {
  RowsArgs a{};
  a.T = T;
  a.features = features;
  a.C = features / B;
  a.B = B;
  a.col_groups = (features + 127) / 128;
  a.groups = (T + 7) / 8 * a.col_groups;
  return a;
}

int expand(const ExpandArgs& e, cudaStream_t s) {
  ExpandKernelArgs a{};
  a.e = e;
  int64_t most = 0;
  for (int i = 0; i < 2; ++i) {
    most = std::max(most, e.gather[i].tiles * e.B * (e.B / 8));
    if (e.rows[i].dst) {
      a.rows[i] = rows_args(e.T, e.rows[i].features, e.B);
      most = std::max(most, a.rows[i].groups * 32);
    }
  }
  if (!most) return BELL_OK;
  unsigned grid;
  if (int rc = grid_for(most, &grid)) return rc;
  bell_mx_expand_kernel<<<grid, kThr, 0, s>>>(a);
  return check_launch("bell_mx_expand_kernel");
}

int finish_grads(const FinishArgs& a, cudaStream_t s) {
  FinishKernelArgs k{a, {}};
  int64_t items = 0, largest = 0;
  for (int i = 0; i < 3; ++i) {
    const TileGrad& g = a.g[i];
    if (g.sums) items += int64_t(g.R) * g.K * g.B * g.B / kFinish;
    k.end[i] = items;
    largest = std::max({largest, items, g.cuts.steps * (int64_t(g.cuts.grid) + 1) + g.cuts.grid});
  }
  if (!items) return BELL_OK;
  unsigned grid;
  if (int rc = grid_for(items * kThr, &grid)) return rc;
  if (largest <= INT32_MAX)
    bell_mx_finish_kernel<uint32_t><<<grid, kThr, 0, s>>>(k);
  else
    bell_mx_finish_kernel<uint64_t><<<grid, kThr, 0, s>>>(k);
  return check_launch("bell_mx_finish_kernel");
}

int add_sums(const float* a, const float* b, int64_t n, void* out, int32_t out_dtype, cudaStream_t s) {
  unsigned grid;
  if (int rc = grid_for(n / 8, &grid)) return rc;
  bell_mx_add_kernel<<<grid, kThr, 0, s>>>(a, b, n, out, out_dtype == BELL_DTYPE_BF16);
  return check_launch("bell_mx_add_kernel");
}

}  // namespace mx
}  // namespace bell

using namespace bell;

extern "C" {

size_t bell_mx_rows_bytes(int64_t T, int32_t features, int32_t B) {
  if (T <= 0 || features <= 0 || (B != 64 && B != 128)) return 0;
  return size_t((T + mx::kRows - 1) / mx::kRows) * size_t(features / B) * size_t(mx::row_chunk(B));
}

size_t bell_mx_tiles_bytes(int32_t R, int32_t K, int32_t B) {
  if (R <= 0 || K <= 0 || (B != 64 && B != 128)) return 0;
  return size_t(R) * size_t(K) * size_t(mx::tile_chunk(B));
}

int bell_mx_quantize_rows(int64_t T, int32_t features, int32_t B, int32_t dtype, const void* src, int64_t ld_src,
                          void* dst, void* stream) {
  if (int rc = mx::check_rows(T, features, B, dtype, src, dst, ld_src)) return rc;
  if (T == 0) return BELL_OK;
  const mx::RowsArgs a = mx::rows_args(T, features, B);
  unsigned grid;
  if (int rc = mx::grid_for(a.groups * 32, &grid)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == BELL_DTYPE_BF16)
    mx::bell_mx_quantize_kernel<<<grid, mx::kThr, 0, s>>>(a, static_cast<const __nv_bfloat16*>(src), ld_src,
                                                          static_cast<uint8_t*>(dst));
  else
    mx::bell_mx_quantize_kernel<<<grid, mx::kThr, 0, s>>>(a, static_cast<const float*>(src), ld_src,
                                                          static_cast<uint8_t*>(dst));
  return check_launch("bell_mx_quantize_rows");
}

int bell_mx_dequantize_rows(int64_t T, int32_t features, int32_t B, const void* src, int32_t dtype, void* dst,
                            int64_t ld_dst, void* stream) {
  if (int rc = mx::check_rows(T, features, B, dtype, dst, src, ld_dst)) return rc;
  if (T == 0) return BELL_OK;
  const mx::RowsArgs a = mx::rows_args(T, features, B);
  unsigned grid;
  if (int rc = mx::grid_for(a.groups * 32, &grid)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint8_t* q = static_cast<const uint8_t*>(src);
  if (dtype == BELL_DTYPE_BF16)
    mx::bell_mx_dequantize_kernel<<<grid, mx::kThr, 0, s>>>(a, q, static_cast<__nv_bfloat16*>(dst), ld_dst);
  else
    mx::bell_mx_dequantize_kernel<<<grid, mx::kThr, 0, s>>>(a, q, static_cast<float*>(dst), ld_dst);
  return check_launch("bell_mx_dequantize_rows");
}

int bell_mx_pack_ell(const BellEll* weights, int32_t n, int32_t dtype, void* const* chunks, void* const* plans,
                     int32_t* status, void* stream) {
  if (!weights || !chunks || !plans) return fail(BELL_ERR_ARG, "bell_mx_pack_ell: NULL argument");
  if (n < 1 || n > BELL_MX_PACK_MAX) return fail(BELL_ERR_ARG, "bell_mx_pack_ell: 1 to BELL_MX_PACK_MAX weights");
  if (dtype != BELL_DTYPE_BF16 && dtype != BELL_DTYPE_F32)
    return fail(BELL_ERR_DTYPE, "bell_mx_pack_ell: dtype must be bf16 or f32");
  mx::PackArgs a{};
  a.n = n;
  int64_t most = 0;
  unsigned plan_end = 0;
  for (int i = 0; i < n; ++i) {
    const BellEll& w = weights[i];
    if (!w.values || !w.col_indices || !chunks[i] || !plans[i]) return fail(BELL_ERR_ARG, "bell_mx_pack_ell: NULL argument");
    if (w.B != 64 && w.B != 128) return fail(BELL_ERR_SHAPE, "bell_mx_pack_ell: tile size B must be 64 or 128");
    if (w.R < 1 || w.C < 1 || w.K < 1) return fail(BELL_ERR_SHAPE, "bell_mx_pack_ell: R, C, K must be >= 1");
    if (w.R > (1 << 23) || w.C > 65535 || w.K > 65535)
      return fail(BELL_ERR_SHAPE, "bell_mx_pack_ell: R must be <= 2^23, C and K <= 65535");
    if (w.layout != BELL_TILE_IN_OUT && w.layout != BELL_TILE_OUT_IN)
      return fail(BELL_ERR_ARG, "bell_mx_pack_ell: unknown tile layout");
    if (!aligned16(w.values) || !aligned16(chunks[i]) || !aligned16(plans[i]))
      return fail(BELL_ERR_ALIGN, "bell_mx_pack_ell: values, chunks and plans must be 16-byte aligned");
    const mx::Plan p = mx::plan_of(plans[i], w.R, w.K);
    const int64_t tiles = int64_t(w.R) * w.K;
    plan_end += unsigned((w.R + mx::kThr / 32 - 1) / (mx::kThr / 32));
    a.w[i] = mx::PackWeight{w.values, tiles, w.B, w.layout == BELL_TILE_IN_OUT, w.col_indices, w.R, w.C, w.K,
                            static_cast<uint8_t*>(chunks[i]), const_cast<uint32_t*>(p.entries),
                            const_cast<int32_t*>(p.counts), plan_end};
    most = std::max(most, tiles * (w.B / 2) * (w.B / mx::kBlock));
  }
  if (int rc = require_sm100()) return rc;
  a.status = status ? status : default_status_ptr();
  if (!a.status) return BELL_ERR_LAUNCH;
  unsigned grid;
  if (int rc = mx::grid_for(most, &grid)) return rc;
  grid += plan_end;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == BELL_DTYPE_BF16)
    mx::bell_mx_pack_kernel<__nv_bfloat16><<<grid, mx::kThr, 0, s>>>(a);
  else
    mx::bell_mx_pack_kernel<float><<<grid, mx::kThr, 0, s>>>(a);
  return check_launch("bell_mx_pack_kernel");
}

int bell_mx_unpack_tiles(const void* chunks0, int64_t tiles0, const void* chunks1, int64_t tiles1, int32_t B,
                         const int64_t* index, int64_t tiles, void* values, void* stream) {
  if (B != 64 && B != 128) return fail(BELL_ERR_SHAPE, "bell_mx_unpack_tiles: tile size B must be 64 or 128");
  if (tiles0 < 0 || tiles1 < 0 || tiles < 0 || (!index && tiles > tiles0 + tiles1))
    return fail(BELL_ERR_SHAPE, "bell_mx_unpack_tiles: bad tile counts");
  if (tiles > 0 && ((tiles0 && !chunks0) || (tiles1 && !chunks1) || !values))
    return fail(BELL_ERR_ARG, "bell_mx_unpack_tiles: NULL buffer");
  if (!aligned16(chunks0) || !aligned16(chunks1) || !aligned16(values))
    return fail(BELL_ERR_ALIGN, "bell_mx_unpack_tiles: buffers must be 16-byte aligned");
  if (int rc = require_sm100()) return rc;
  if (tiles == 0) return BELL_OK;
  unsigned grid;
  if (int rc = mx::grid_for(tiles * B * (B / 8), &grid)) return rc;
  mx::bell_mx_unpack_kernel<<<grid, mx::kThr, 0, static_cast<cudaStream_t>(stream)>>>(
      mx::TileGather{chunks0, tiles0, chunks1, tiles1, index, tiles, values}, B);
  return check_launch("bell_mx_unpack_kernel");
}

}  // extern "C"
