// Device code shared by the kernels on 4-bit rows (gf_mx*.hip).
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <type_traits>

#include "gf_operators.h"

namespace gf {
namespace {

template <int DT>
struct Elem;
template <>
struct Elem<GF_F32> {
    using T = float;
};
template <>
struct Elem<GF_F16> {
    using T = _Float16;
};
template <>
struct Elem<GF_BF16> {
    using T = __bf16;
};
template <int DT>
using ElemT = typename Elem<DT>::T;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// 2^(byte - 127); byte 0 is the subnormal 2^-127, byte 255 NaN.
__device__ __forceinline__ float mx_scale(uint32_t byte) {
    return __uint_as_float(byte == 255u ? 0x7FC00000u : byte ? byte << 23 : 1u << 22);
}

// 16 bytes at an address aligned to an element only.
struct __attribute__((packed, aligned(1))) Bytes16 {
    uint4 v;
};
__device__ __forceinline__ uint4 load16(const void* p) { return static_cast<const Bytes16*>(p)->v; }
// The same for what is read once.
__device__ __forceinline__ uint4 load16_once(const void* p) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(1)));
    const u32x4 v = __builtin_nontemporal_load(static_cast<const u32x4*>(p));
    return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store16(void* p, uint4 v) { static_cast<Bytes16*>(p)->v = v; }

// Workgroups go to the eight XCDs in turn, each with an L2 of its own: ids are
// dealt so that an XCD works on a run of consecutive tiles.
__device__ __forceinline__ uint32_t xcd_run(uint32_t b, uint32_t n) {
    const uint32_t x = b & 7u, per = n >> 3, rem = n & 7u;
    return x * per + min(x, rem) + (b >> 3);
}
// Tile t of a grid of tm x tn, in bands of `band` rows of tiles, each walked
// column by column: the tiles in flight share rows of both operands.
__device__ __forceinline__ void tile_of(uint32_t t, uint32_t tm, uint32_t tn, uint32_t band, uint32_t& m, uint32_t& n) {
    const uint32_t per = band * tn, g = t / per, r = t % per, h = min(band, tm - g * band);
    m = g * band + r % h;
    n = r / h;
}

// A wave's 32 x COLS piece of a result, from four consecutive columns a lane
// (put: row, column, four values) to 16-byte stores of whole rows, through
// kBytes of LDS that only this wave uses.
template <int OT, uint32_t COLS>
struct Piece {
    using T = ElemT<OT>;
    static constexpr uint32_t kPitch = COLS * sizeof(T) + 16u;
    static constexpr uint32_t kBytes = 32u * kPitch;
    static __device__ __forceinline__ void put(uint8_t* lds, uint32_t row, uint32_t col, f32x4 v) {
        T* p = reinterpret_cast<T*>(lds + row * kPitch) + col;
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 o;
        for (int i = 0; i < 4; ++i) o[i] = T(v[i]);
        *reinterpret_cast<T4*>(p) = o;
    }
    // Rows m0.. and columns n0.. of out, M x N.
    static __device__ __forceinline__ void flush(const uint8_t* lds, T* out, uint64_t ldo, uint32_t m0, uint32_t n0,
                                                 uint32_t M, uint32_t N) {
        constexpr uint32_t V = 16u / sizeof(T), per = COLS / V, kTurns = per / 2u;   // elements a store, stores a row
        const uint32_t lane = threadIdx.x & 63u;
        if (m0 + 32u <= M && n0 + COLS <= N) {
            const uint32_t c = lane % per * V, r = lane / per;
            T* p = out + uint64_t(m0 + r) * ldo + n0 + c;
            uint4 v[kTurns];
#pragma unroll
            for (uint32_t i = 0; i < kTurns; ++i)
                v[i] = *reinterpret_cast<const uint4*>(lds + (r + i * (64u / per)) * kPitch + c * sizeof(T));
#pragma unroll
            for (uint32_t i = 0; i < kTurns; ++i) store16(p + uint64_t(i * (64u / per)) * ldo, v[i]);
        } else {
            const uint32_t c = lane % COLS;
            if (n0 + c < N)
                for (uint32_t r = lane / COLS; r < 32u && m0 + r < M; r += 64u / COLS)
                    out[uint64_t(m0 + r) * ldo + n0 + c] = reinterpret_cast<const T*>(lds + r * kPitch)[c];
        }
    }
};
// LDS byte address of a __shared__ object.
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return uint32_t(uintptr_t((const __attribute__((address_space(3))) void*)p));
}
// Asynchronous global-to-LDS copies: 16 bytes per active lane from base + off
// (base wave-uniform) to LDS at lds_base + 16 x lane, lds_base wave-uniform
// (in m0).  They count in vmcnt and the compiler does not see them (for copies
// that it sees it waits before any LDS read): the caller waits (wait_vmcnt)
// and synchronises before the data is read.
__device__ __forceinline__ void lds_copy16(const uint8_t* base, uint32_t off, uint32_t lds_base) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(lds_base) : "memory");
}
// s_waitcnt vmcnt(N), the other counters unconstrained (gfx9 encoding).
template <uint32_t N>
__device__ __forceinline__ void wait_vmcnt() {
    static_assert(N < 64u, "vmcnt");
    __builtin_amdgcn_s_waitcnt(int((N & 15u) | ((N >> 4) << 14) | (7u << 4) | (15u << 8)));
}
// No instruction is scheduled across this point.
__device__ __forceinline__ void sched_fence() { __builtin_amdgcn_sched_barrier(0); }
// A barrier behind this wave's LDS accesses; it waits for no global ones.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// Orders a wave's own LDS writes before its reads by other lanes.
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Compute units of the current device.
inline uint32_t compute_units() {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
        return 256u;
    return uint32_t(n);
}

// Whether a result of M x N is better cut into tiles of 256 than of 128.  A
// compute unit holds one of the large or two of the small ones, and a large one
// takes as long as two rounds of small ones at most: so where it does not take
// more rounds.  Large against small: 8192 x 8192 x 4096 187 us
// against 250, 4096 x 4096 x 2048 26 against 30, 1000 x 4096 x 4096 32 against
// 18, 1000 x 20000 x 768 23 against 20.
inline bool large_tiles(uint64_t M, uint64_t N, uint64_t cus) {
    const uint64_t big = ((M + 255u) / 256u) * ((N + 255u) / 256u), small = ((M + 127u) / 128u) * ((N + 127u) / 128u);
    return 2u * ((big + cus - 1u) / cus) <= (small + 2u * cus - 1u) / (2u * cus);
}

template <class F>
hipError_t by_type(int32_t dtype, F&& f) {
    if (dtype == GF_F32) return f(std::integral_constant<int, GF_F32>());
    if (dtype == GF_F16) return f(std::integral_constant<int, GF_F16>());
    return f(std::integral_constant<int, GF_BF16>());
}

}  // namespace
}  // namespace gf
