// Device helpers of the cache kernels: lengths and pages with their bounds, e4m3 conversions, the f16 tensor instructions.
#pragma once
#include <cuda_fp16.h>
#include "dm_cache.h"
#include "dm_common.cuh"

namespace dm {

// What the host cannot see without a synchronisation is checked here: a bad value is reported through the status word and replaced by one
// that keeps every access inside the buffers.
__device__ __forceinline__ void report(int* status, int code) {
  if (status != nullptr) {
    volatile int* s = status;
    if (*s == 0) *s = code;
  }
}
__device__ __forceinline__ int cache_length(const CacheView& c, int b) {
  const int n = __ldg(c.lengths + b), cap = c.T * c.page;
  if (n < 0 || n > cap) {
    report(c.status, kStatusBadLength + kInCache);
    return n < 0 ? 0 : cap;
  }
  return n;
}
__device__ __forceinline__ int checked_page(const CacheView& c, int id) {
  if (static_cast<unsigned>(id) >= static_cast<unsigned>(c.pages)) {
    report(c.status, kStatusBadPage + kInCache);
    return -1;
  }
  return id;
}
__device__ __forceinline__ int checked_count(int* status, const int* counts, int b, int most) {
  if (counts == nullptr) return most;
  const int n = __ldg(counts + b);
  if (n < 0 || n > most) {
    report(status, kStatusBadLength + kInCache);
    return n < 0 ? 0 : most;
  }
  return n;
}

// Two e4m3 codes (low 16 bits / high 16 bits of a word) -> two f16 values, exact.
__device__ __forceinline__ uint32_t e4m3_lo_f16x2(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_hi_f16x2(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ float2 f16x2_to_float2(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Four codes times a power of two -> four codes (round to nearest even).
__device__ __forceinline__ uint32_t requant4(uint32_t w, float ratio) {
  const float2 a = f16x2_to_float2(e4m3_lo_f16x2(w)), b = f16x2_to_float2(e4m3_hi_f16x2(w));
  return cvt_e4m3x4(a.x * ratio, a.y * ratio, b.x * ratio, b.y * ratio);
}

// Below all logits: a row's reference before the first one (infinities would not cancel).
constexpr float kNone = -3e38f;

// 0xFF in the bytes of four e4m3 codes that are NaN.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu); }

// Four 8 x 16-byte matrices; lane l gives the address of row l % 8 of matrix l / 8.  Thread (g = lane / 4, t = lane % 4) receives bytes
// 4 t ... 4 t + 3 of row g of each.
__device__ __forceinline__ void ldmatrix4(uint32_t saddr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(saddr) : "memory");
}
// The same, transposed in pairs of bytes: bytes 2 g, 2 g + 1 of row 2 t, then of row 2 t + 1.
__device__ __forceinline__ void ldmatrix4_trans(uint32_t saddr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(saddr) : "memory");
}
// 8 x 8 f16 matrix across the warp, transposed.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
// D (16 x 8 fp32) += A (16 x 16 f16) B (16 x 8 f16).
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}

// 4-D tiled load: coordinates innermost first, x * element size a multiple of 16 bytes.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

}  // namespace dm
