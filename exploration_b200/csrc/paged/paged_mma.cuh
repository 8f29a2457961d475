// Warp-level matrix instructions of the few-row kernel, 16-bit packing and range
// of the weights, and the tcgen05 instruction descriptor of the chunk kernel.
#pragma once

#include <type_traits>

#include "../common/sm100.cuh"

namespace eb {
namespace paged {

EB_DEVICE void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

EB_DEVICE void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// d += a b, a [16 rows x 16], b [16 x 8], fp32 accumulation.
template <typename T>
EB_DEVICE void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

template <typename T>
EB_DEVICE uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// Weights are rounded to the input type for the second product, and fp16 keeps 11 bits
// down to 2^-14 only: relative to a largest weight of one, a key 2^-25 below it would
// vanish, however many there are. Reference points therefore lie below the maximum so
// that the largest weight is 2^kWeightExp; sums and partial results carry the same
// factor, which cancels. bf16 has the range of fp32. Rounding a reference point
// up keeps the largest weight from passing that power at logits beyond 2^24.
template <typename T>
constexpr float kWeightExp = std::is_same_v<T, __half> ? 15.f : 0.f;

// Reference point of a row whose largest score is `top`, `below` the maximum (log2 units).
EB_DEVICE float reference_point(float top, float scale_log2, float below) { return __fmaf_ru(top, scale_log2, -below); }

// Bounded wait of the tile loops: sm100::mbar_wait without its sleep between
// polls (the poll itself suspends the warp for a while); the time and the abort
// word are looked at every 32 polls.
EB_DEVICE bool wait_tight(uint64_t* bar, uint32_t parity, volatile int* abort, sm100::ErrorSlot* err, int site) {
  if (sm100::mbar_try_wait(bar, parity)) return true;
  const long long start = clock64();
  for (int i = 1;; ++i) {
    if (sm100::mbar_try_wait(bar, parity)) return true;
    if ((i & 31) == 0) {
      if (*abort) return false;
      if (clock64() - start > 2000000000LL) {   // about a second
        *abort = 1;
        sm100::report(err, site);
        return false;
      }
    }
  }
}

// Three-input maximum and two-wide fp32 arithmetic of sm_100.
EB_DEVICE float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

EB_DEVICE float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

EB_DEVICE float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Instruction descriptor of kind::f16 with both operands fp16 or both bf16, fp32 accumulation.
EB_HOST_DEVICE uint32_t idesc_16(bool bf16, int m, int n, bool a_mn_major, bool b_mn_major) {
  const uint32_t type = bf16 ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | (static_cast<uint32_t>(a_mn_major) << 15) |
         (static_cast<uint32_t>(b_mn_major) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

}  // namespace paged
}  // namespace eb
