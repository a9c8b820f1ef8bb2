// bell_mx.cuh — the MXFP4 layouts (e2m1 codes with one e8m0 scale for 32
// values along the contraction) and the device helpers that read and write them.
//
// Everything is stored in the form the tensor core consumes, so that operands
// move with untiled bulk copies and no kernel shuffles nibbles:
//
//   atom   N rows x 64 values (32 bytes a row) as 8-row x 16-byte core
//          matrices: byte b of row n at (n/8)*256 + (b/16)*128 + (n%8)*16 + b%16
//          (K-major without swizzle: LBO 128, SBO 256).  Value 2i of a row is
//          the low nibble of byte i.  One atom is the K = 64 of one MMA.
//   scales 512 bytes: scale j (0..3) of row n at (n%32)*16 + (n/32)*4 + j,
//          the image of tcgen05.cp.32x128b (four 32-bit TMEM columns of 32
//          lanes).
//   chunk  B/64 atoms, then the scales: the activations' [128 tokens x B]
//          piece or the weights' [B outputs x B inputs] tile.
//
// Rows:  chunk (m, c) at (m * C + c) * row_chunk(B): tokens 128m.. of column
//        block c.  Rows past the last token are never written nor used.
// Tiles: chunk (r, k) at (r * K + k) * tile_chunk(B).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "bell_host.h"
#include "bell_ptx.cuh"

namespace bell {
namespace mx {

static constexpr int kRows = 128;       // tokens of a chunk (MMA M)
static constexpr int kBlock = 32;       // values of one scale
static constexpr int kScaleBytes = 512;

__host__ __device__ constexpr int row_chunk(int B) { return kRows * B / 2 + kScaleBytes; }
__host__ __device__ constexpr int tile_chunk(int B) { return B * B / 2 + kScaleBytes; }

// Offset of the 16 bytes holding scale block j (32 values) of row n of a
// chunk whose atoms are `atom` bytes (32 x rows).
__host__ __device__ constexpr int code_off(int n, int j, int atom) {
  return (j >> 1) * atom + (n >> 3) * 256 + (j & 1) * 128 + (n & 7) * 16;
}
__host__ __device__ constexpr int scale_off(int n, int j) { return (n & 31) * 16 + (n >> 5) * 4 + j; }

// Scale byte of a block whose largest magnitude has the fp32 bits `top`:
// exponent floor(log2 top) - 2, not below 2^-127; 255 when it is not finite.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// 1 / scale, exact (2^127 .. 2^-125); a non-finite block has no finite codes,
// any multiplier does.
__device__ __forceinline__ float scale_inverse(uint32_t byte) {
  return __uint_as_float((byte == 255u ? 127u : 254u - byte) << 23);
}
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7FC00000u : (byte ? byte << 23 : 0x00400000u));
}

// Eight e2m1 codes, round to nearest even, saturating at 6; v[0] lowest.
__device__ __forceinline__ uint32_t pack_e2m1(const float* v) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Raise the transaction count of the current phase without arriving.
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

// 32 bytes of one thread: a whole sector of global memory (p 32-byte aligned).
__device__ __forceinline__ void st_global_v8(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void ld_global_v8(const void* p, uint32_t (&v)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "l"(p)
               : "memory");
}

// Two fp32 products or sums in one instruction, each rounded as alone.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
// Largest magnitude of three; NaN if one is.
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// One scale block: codes of v[0..31] and the scale byte.
__device__ __forceinline__ uint4 quantize32(const float (&v)[32], uint32_t& byte) {
  float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = max_abs3(m[j], v[i + 2 * j], v[i + 2 * j + 1]);
  }
  const float top = max_abs3(max_abs3(m[0], m[1], m[2]), m[3], 0.f);
  byte = scale_byte(__float_as_uint(top) & 0x7FFFFFFFu);
  const float inv = scale_inverse(byte);
  float s[32];
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    const float2 t = mul2(make_float2(v[i], v[i + 1]), make_float2(inv, inv));
    s[i] = t.x;
    s[i + 1] = t.y;
  }
  return make_uint4(pack_e2m1(s), pack_e2m1(s + 8), pack_e2m1(s + 16), pack_e2m1(s + 24));
}

// Eight codes -> values times the scale.
__device__ __forceinline__ void unpack_e2m1(uint32_t w, float scale, float* v) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h[i]));
    v[2 * i] = f.x * scale;
    v[2 * i + 1] = f.y * scale;
  }
}

// 32 consecutive values of a row, 16-byte loads.
__device__ __forceinline__ void load32(const __nv_bfloat16* p, float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 w = ld_global_nc_v4(p + 8 * i);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack_bf16x2(u[j]);
      v[8 * i + 2 * j] = f.x;
      v[8 * i + 2 * j + 1] = f.y;
    }
  }
}
__device__ __forceinline__ void load32(const float* p, float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint4 w = ld_global_nc_v4(p + 4 * i);
    v[4 * i] = __uint_as_float(w.x);
    v[4 * i + 1] = __uint_as_float(w.y);
    v[4 * i + 2] = __uint_as_float(w.z);
    v[4 * i + 3] = __uint_as_float(w.w);
  }
}
// ------------------------------------------------------------------ tcgen05

// Shared-memory matrix descriptors without swizzle, as two words: the low one
// (start address and LBO, in 16-byte units) moves with the stage, the high one
// (SBO and the version) is a constant.  They are joined inside the
// instructions' asm, so that no 64-bit arithmetic is done on descriptors.
__device__ __forceinline__ uint32_t sdesc_lo(uint32_t saddr, uint32_t lbo) {
  return ((saddr >> 4) & 0x3FFFu) | ((lbo >> 4) << 16);
}
static constexpr uint32_t kOperandHi = (256u >> 4) | (1u << 14);  // 8-row groups 256 bytes apart
static constexpr uint32_t kScaleHi = (128u >> 4) | (1u << 14);    // 8 x 16 bytes after 8 x 16 bytes

// kind::mxf4 instruction descriptor: e2m1 x e2m1 -> f32, ue8m0 scales; both
// operands K-major; sf selects scale bytes (0: the first two of a 32-bit
// column, 2: the last two) for both.
__host__ __device__ constexpr uint32_t idesc_mxf4(int M, int N, uint32_t sf) {
  return (sf << 4) | (1u << 7) | (1u << 10) | (uint32_t(N >> 3) << 17) | (1u << 23) | (uint32_t(M >> 7) << 27) |
         (sf << 29);
}

// D[tmem] (+)= A x B over K = 64, A and B from shared memory (low descriptor
// words), scales in TMEM.
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t sfa,
                                         uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 da, {%1, %7};\n\t"
      "mov.b64 db, {%2, %7};\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], da, db, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(kOperandHi)
      : "memory");
}

// Scales: 32 x 16 bytes of shared memory into four TMEM columns, repeated in
// each quarter of the lanes.  Runs in order with this thread's later MMAs.
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t desc) {
  asm volatile(
      "{\n\t.reg .b64 ds;\n\t"
      "mov.b64 ds, {%1, %2};\n\t"
      "tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], ds;\n\t}\n" ::"r"(tmem), "r"(desc), "r"(kScaleHi)
      : "memory");
}

// 16 columns at ta and 16 at tb of this warp's 32 lanes, and the wait.
__device__ __forceinline__ void tmem_ld16x2_sync(uint32_t ta, uint32_t (&a)[16], uint32_t tb, uint32_t (&b)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]), "=r"(a[8]), "=r"(a[9]), "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15]), "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]), "=r"(b[4]), "=r"(b[5]), "=r"(b[6]), "=r"(b[7]), "=r"(b[8]), "=r"(b[9]), "=r"(b[10]), "=r"(b[11]), "=r"(b[12]), "=r"(b[13]), "=r"(b[14]), "=r"(b[15])
      : "r"(ta), "r"(tb)
      : "memory");
}

// ------------------------------------------------------------- weight plan

// Live slots of each block-row in ascending slot order (entry = column |
// slot << 16), then kNoSlot up to K; and their number.  [R, K] entries, then
// [R] counts, each part padded to 16 bytes (bell_plan_bytes(0, 0, 0, R, K)
// bytes).
static constexpr uint32_t kNoSlot = 0xFFFFFFFFu;  // column and slot are at most 65534
struct Plan {
  const uint32_t* entries;
  const int32_t* counts;
};
inline Plan plan_of(const void* plan, int32_t R, int32_t K) {
  const PlanLayout L = plan_layout(0, 0, 0, R, K);
  const char* p = static_cast<const char*>(plan);
  return {reinterpret_cast<const uint32_t*>(p + L.d_entries), reinterpret_cast<const int32_t*>(p + L.d_counts)};
}

// Gathered tiles to bf16 [tiles, B_out, B_in]: tile index[i] (or i) of the n0
// tiles at c0 followed by the n1 at c1.
struct TileGather {
  const void* c0;
  int64_t n0;
  const void* c1;
  int64_t n1;
  const int64_t* index;
  int64_t tiles;
  void* values;
};
struct RowsTo {  // quantised rows to bf16 [T, features]
  const void* src;
  int32_t features;
  void* dst;
};
// Everything that a backward unpacks before its products, one launch.
struct ExpandArgs {
  int64_t T;
  int32_t B;
  TileGather gather[2];
  RowsTo rows[2];
};
int expand(const ExpandArgs& e, cudaStream_t s);
// A tile gradient [R, K, B, B]: its sums as sddmm_bf16 leaves them
// (bell_host.h), completed by the parts of their units, zero in dead slots, and,
// where `rounded` is given, written there in bf16.
struct TileGrad {
  float* sums;
  void* rounded;
  const float* parts;   // optional
  const int32_t* cols;  // [R, K]: live in [0, C), C = 0 without tokens
  int32_t R, C, K, B;
  SddmmCuts cuts;
};
struct FinishArgs {
  TileGrad g[3];  // without sums: skipped
};
int finish_grads(const FinishArgs& a, cudaStream_t s);
// out = a + b, n fp32 values (a multiple of 8); out fp32 (a itself may be) or bf16.
int add_sums(const float* a, const float* b, int64_t n, void* out, int32_t out_dtype, cudaStream_t s);

// [d_gate | d_up] (bf16 [T, 2 R B]) from d_h (fp32 [T, R B]) and the gated
// block's quantised rows and weights (bell_mx.cu).
int gated_backward(int64_t T, const void* x, const BellMxEll& gate, const BellMxEll& up, const float* dh, void* dgu,
                   int32_t* status, cudaStream_t s);

// Argument checks of rows [T, features], ld elements apart (bell_mx_quant.cu).
int check_rows(int64_t T, int32_t features, int32_t B, int32_t dtype, const void* rows, const void* chunks, int64_t ld);

}  // namespace mx
}  // namespace bell
