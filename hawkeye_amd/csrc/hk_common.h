// Shared device/host helpers for the gfx950 kernels (wave64, MFMA, LDS-DMA).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include "../../include/hawkeye_hip.h"
#include <atomic>

// Once per (kernel instantiation, device): hipFuncSetAttribute acts on the CURRENT device's copy of the function, and one
// process may drive two devices (the two-device placement of set_device_ids).  `done` is a per-instantiation bit mask of
// the devices already set up; racing first calls set the same value.  Returns hipSuccess or the failing call's error.
static inline hipError_t hk_lds_attr_once(std::atomic<unsigned long long>& done, const void* func, int lds_bytes) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    if (dev < 0 || dev >= 64) return hipErrorInvalidDevice;
    if ((done.load(std::memory_order_acquire) >> dev) & 1ull) return hipSuccess;
    e = hipFuncSetAttribute(func, hipFuncAttributeMaxDynamicSharedMemorySize, lds_bytes);
    if (e == hipSuccess) done.fetch_or(1ull << dev, std::memory_order_release);
    return e;
}

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

#define HK_LOG2E 1.4426950408889634f

// fp32 -> bf16 with round-to-nearest-even; hipcc lowers the cast to v_cvt_pk_bf16_f32 on gfx950.
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
    bf16x2 v;
    v[0] = (__bf16)lo;
    v[1] = (__bf16)hi;
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }

// LDS-DMA: 16 bytes per lane, destination = wave-uniform LDS base + lane * 16.
__device__ __forceinline__ void glds16(const void* gsrc, void* lds_wave_base) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)gsrc,
                                     (__attribute__((address_space(3))) void*)lds_wave_base, 16, 0, 0);
}

// LDS-DMA with a scalar base: address = SGPR pair + one 32-bit per-lane byte offset (no 64-bit vector address
// arithmetic per piece).  Inline asm: the builtin always takes a 64-bit vector address.  lds = the wave's destination.
__device__ __forceinline__ void glds16_s(const void* sbase, uint32_t voff, const void* lds) {
    const uint32_t la = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)lds;
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :
                 : "v"(voff), "s"(sbase), "s"(la)
                 : "memory");
}
// The same with a 64-bit per-lane address.  A kernel that uses these helpers issues EVERY LDS-DMA through them, so the
// compiler itself never holds a value in M0 there (M0 is reserved and cannot be named as a clobber), and retires them with
// its own counted s_waitcnt vmcnt (the compiler does not know these statements write LDS).
__device__ __forceinline__ void glds16_v(const void* vaddr, const void* lds) {
    const uint32_t la = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)lds;
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                 :
                 : "v"(vaddr), "s"(la)
                 : "memory");
}

// 4 bytes per lane (256 B per wave-instruction), scalar base + 32-bit lane offset.
__device__ __forceinline__ void glds4_s(const void* sbase, uint32_t voff, const void* lds) {
    const uint32_t la = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)lds;
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
                 :
                 : "v"(voff), "s"(sbase), "s"(la)
                 : "memory");
}

void hk_set_error(const char* fmt, ...);

// Host-side check that what a call writes shares no byte with what it reads: an operand of n1 x n2 rows of `row` elements (strides in
// elements, not negative), from its first byte a to the one behind its last, b.  A null operand has no rows.
struct HkSpan {
    uintptr_t a, b;
    int64_t n1, s1, n2, s2, row;     // in bytes
};
static inline HkSpan hk_span(const void* ptr, int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t row, int64_t elem) {
    if (!ptr || n1 < 1 || n2 < 1 || row < 1) return {};
    const uintptr_t a = reinterpret_cast<uintptr_t>(ptr);
    return {a, a + (uintptr_t)(((n1 - 1) * s1 + (n2 - 1) * s2 + row) * elem), n1, s1 * elem, n2, s2 * elem, row * elem};
}
// Pieces of x and y that begin at a + (whole multiples of g) and are px and py bytes long never meet if they lie side by side within g.
static inline bool hk_side_by_side(uintptr_t xa, int64_t px, uintptr_t ya, int64_t py, uint64_t g) {
    if (g == 0) return false;
    const uint64_t d = ya >= xa ? (ya - xa) % g : (g - (xa - ya) % g) % g;      // y's place within x's period
    return d >= (uint64_t)px && d + (uint64_t)py <= g;
}
// Operands interleaved in one tensor (K and V of a cache [B, rows, 2, H, hd] or [B, 2, rows, H, hd]) do not overlap, though their spans do: rows,
// or the whole blocks that one index leaves, lie side by side.  May find an overlap where a layout is more intricate than that, never the reverse.
static inline bool hk_overlap(const HkSpan& x, const HkSpan& y) {
    if (x.a >= y.b || y.a >= x.b) return false;
    auto gcd = [](int64_t p, int64_t q) {
        while (q) {
            const int64_t r = p % q;
            p = q;
            q = r;
        }
        return p;
    };
    const int64_t g1 = gcd(x.n1 > 1 ? x.s1 : 0, y.n1 > 1 ? y.s1 : 0), g2 = gcd(x.n2 > 1 ? x.s2 : 0, y.n2 > 1 ? y.s2 : 0);
    return !hk_side_by_side(x.a, x.row, y.a, y.row, gcd(g1, g2)) &&
           !hk_side_by_side(x.a, (x.n2 - 1) * x.s2 + x.row, y.a, (y.n2 - 1) * y.s2 + y.row, g1) &&
           !hk_side_by_side(x.a, (x.n1 - 1) * x.s1 + x.row, y.a, (y.n1 - 1) * y.s1 + y.row, g2);
}

// Rows of `row` elements at i1 * s1 + i2 * s2 (i1 < n1, i2 < n2) that a call writes: no two share an element, the one index within the other's steps.
static inline bool hk_rows_apart(int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t row) {
    if ((n1 > 1 && s1 < row) || (n2 > 1 && s2 < row)) return false;
    return n1 <= 1 || n2 <= 1 || s1 >= (n2 - 1) * s2 + row || s2 >= (n1 - 1) * s1 + row;
}

#define HK_REQUIRE(cond, ...)            \
    do {                                 \
        if (!(cond)) {                   \
            hk_set_error(__VA_ARGS__);   \
            return HK_EINVAL;            \
        }                                \
    } while (0)

#define HK_CHECK_LAUNCH(name)                                               \
    do {                                                                    \
        hipError_t e_ = hipGetLastError();                                  \
        if (e_ != hipSuccess) {                                             \
            hk_set_error("%s: launch failed: %s", name, hipGetErrorString(e_)); \
            return HK_ELAUNCH;                                              \
        }                                                                   \
    } while (0)
