// Rows in microscaled 4-bit floating point: quantisation, products, gradient
// (gfx950, wave64).  The format and its layout are described at gf_mx_rows.
#include <algorithm>

#include "gf_mx_device.h"

namespace gf {
namespace {

// ---- quantisation ---------------------------------------------------------
// Both directions are bound by memory.  A lane holds 16 bytes of the real side
// (V = 4 or 8 values), so 8 or 4 lanes share a block and 32 or 16 a chunk of
// 128 values; kAhead chunks a lane are loaded before the first is used.  1M x
// 128: fp32 96 us to codes (6.1 TB/s; 105 with loads that stay in the caches),
// bfloat16 52 us (61 with one chunk ahead); back in turn with quantisations 115 and
// 90 us (141 and 92 with one chunk ahead, 115 and 99 with four), by itself 148 and
// 85, binary16 87: 3.7 to 3.9 TB/s, where a fill of the same bytes takes 78 and 40.
// Rows that are not whole chunks of 16-byte pieces share lines: 1M x 130 235 us in
// fp32, 2.8 TB/s, 135 in bfloat16.

template <bool BACK>
constexpr uint32_t kAhead = BACK ? 2 : 4;

// The scale byte of a block whose magnitudes' largest bit pattern (fp32) is
// top: floor(log2) is the exponent field - 127 (a subnormal's is below the
// least scale anyway), 2 less for the grid's largest binade.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
    const uint32_t e = top >> 23;
    return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}

// Chunks (row, s) of a grid-strided walk; the division by S is done once.
struct Walk {
    uint64_t row;
    uint32_t s;
    uint64_t drow;
    uint32_t ds, S;
    __device__ __forceinline__ Walk(uint64_t first, uint64_t step, uint32_t chunks) : S(chunks) {
        row = first / S, s = uint32_t(first % S);
        drow = step / S, ds = uint32_t(step % S);
    }
    __device__ __forceinline__ void next() {
        row += drow, s += ds;
        if (s >= S) s -= S, ++row;
    }
};

template <int DT>
__global__ __launch_bounds__(256) void k_mx_quantise(const ElemT<DT>* x, uint64_t rows, uint32_t K, uint64_t ld, uint32_t S,
                                                     uint8_t* codes, uint8_t* scales) {
    using T = ElemT<DT>;
    constexpr uint32_t V = 16u / sizeof(T), kLanes = 128u / V, kChunks = 256u / kLanes;
    const uint32_t lane = threadIdx.x % kLanes;
    Walk at(uint64_t(blockIdx.x) * kChunks + threadIdx.x / kLanes, uint64_t(gridDim.x) * kChunks, S);
    while (at.row < rows) {   // a chunk's lanes agree on this
        uint4 raw[kAhead<false>];
        Walk w = at;
#pragma unroll
        for (uint32_t u = 0; u < kAhead<false>; ++u, w.next()) {
            const uint32_t k = w.s * 128u + lane * V;
            raw[u] = make_uint4(0, 0, 0, 0);
            if (w.row >= rows) continue;
            const T* p = x + w.row * ld + k;
            if (k + V <= K) {
                raw[u] = load16_once(p);
            } else {
                T t[V];
#pragma unroll
                for (uint32_t i = 0; i < V; ++i) t[i] = k + i < K ? p[i] : T(0.0f);
                __builtin_memcpy(&raw[u], t, 16);
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < kAhead<false>; ++u, at.next()) {
            T t[V];
            __builtin_memcpy(t, &raw[u], 16);
            float v[V];
            uint32_t top = 0;
            if constexpr (DT == GF_BF16) {   // the upper halves of fp32 bit patterns, two a word
                typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
                u16x2 m = {0, 0};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t word = (&raw[u].x)[i] & 0x7FFF7FFFu;
                    u16x2 h;
                    __builtin_memcpy(&h, &word, 4);
                    m = __builtin_elementwise_max(m, h);
                }
                top = uint32_t(max(m[0], m[1])) << 16;
            } else {
#pragma unroll
                for (uint32_t i = 0; i < V; ++i) {
                    v[i] = float(t[i]);
                    top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
                }
            }
            top = max(top, uint32_t(__builtin_amdgcn_mov_dpp(int(top), 0xB1, 0xF, 0xF, true)));   // lane ^ 1
            top = max(top, uint32_t(__builtin_amdgcn_mov_dpp(int(top), 0x4E, 0xF, 0xF, true)));   // lane ^ 2
            if (V == 4) top = max(top, uint32_t(__builtin_amdgcn_mov_dpp(int(top), 0x141, 0xF, 0xF, true)));   // 7 - lane
            const uint32_t byte = scale_byte(top);
            const float scale = mx_scale(byte == 255u ? 127u : byte);
            uint32_t c = 0;
            if constexpr (DT == GF_BF16) {
                bf16x2 p[4];
                __builtin_memcpy(p, &raw[u], 16);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, p[0], scale, 0);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, p[1], scale, 1);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, p[2], scale, 2);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, p[3], scale, 3);
            } else {
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
            }
            if constexpr (DT == GF_F16) {
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
            }
            if (byte == 255u) c = 0;
            if (at.row >= rows) continue;
            const uint64_t chunk = at.row * S + at.s;
            if constexpr (V == 8)
                reinterpret_cast<uint32_t*>(codes)[chunk * 16u + lane] = c;
            else
                reinterpret_cast<uint16_t*>(codes)[chunk * 32u + lane] = uint16_t(c);
            if (lane % (32u / V) == 0) scales[chunk * 4u + lane / (32u / V)] = uint8_t(byte);
        }
    }
}

template <int DT>
__global__ __launch_bounds__(256) void k_mx_dequantise(gf_mx_rows w, uint32_t S, ElemT<DT>* out, uint64_t ld) {
    using T = ElemT<DT>;
    constexpr uint32_t V = 16u / sizeof(T), kLanes = 128u / V, kChunks = 256u / kLanes;
    const uint32_t lane = threadIdx.x % kLanes;
    Walk at(uint64_t(blockIdx.x) * kChunks + threadIdx.x / kLanes, uint64_t(gridDim.x) * kChunks, S);
    while (at.row < w.rows) {
        uint32_t c[kAhead<true>], sc[kAhead<true>];
        Walk a = at;
#pragma unroll
        for (uint32_t u = 0; u < kAhead<true>; ++u, a.next()) {
            const uint64_t chunk = min(a.row, w.rows - 1u) * S + a.s;
            if constexpr (V == 8)
                c[u] = reinterpret_cast<const uint32_t*>(w.codes)[chunk * 16u + lane];
            else
                c[u] = reinterpret_cast<const uint16_t*>(w.codes)[chunk * 32u + lane];
            sc[u] = w.scales[chunk * 4u + lane / (32u / V)];
        }
#pragma unroll
        for (uint32_t u = 0; u < kAhead<true>; ++u, at.next()) {
            if (at.row >= w.rows) continue;
            const float scale = mx_scale(sc[u]);
            T t[V];
            auto two = [&](uint32_t i, auto sel) {
                if constexpr (DT == GF_BF16) {
                    const bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[u], scale, decltype(sel)::value);
                    t[i] = p[0], t[i + 1] = p[1];
                } else {
                    const f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], scale, decltype(sel)::value);
                    t[i] = T(p[0]), t[i + 1] = T(p[1]);
                }
            };
            two(0, std::integral_constant<int, 0>());
            two(2, std::integral_constant<int, 1>());
            if constexpr (V == 8) {
                two(4, std::integral_constant<int, 2>());
                two(6, std::integral_constant<int, 3>());
            }
            const uint32_t k = at.s * 128u + lane * V;
            T* p = out + at.row * ld + k;
            if (k + V <= w.K) {
                uint4 q;
                __builtin_memcpy(&q, t, 16);
                store16(p, q);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < V; ++i)
                    if (k + i < w.K) p[i] = t[i];
            }
        }
    }
}

}  // namespace

namespace {
// Workgroups for a walk over rows x S chunks, 256 threads of `ahead` 16-byte
// pieces each: one turn where they fit the grid.
uint32_t walk_blocks(uint64_t rows, uint32_t S, uint32_t elem, uint32_t ahead) {
    const uint64_t per = 256u / (128u * elem / 16u) * ahead;
    return uint32_t(std::min<uint64_t>((rows * S + per - 1u) / per, 1u << 20));
}
}  // namespace

hipError_t launch_mx_quantise(const MatIn& x, uint32_t K, uint8_t* codes, uint8_t* scales, hipStream_t st) {
    const uint32_t S = mx_chunks(K);
    return by_type(x.dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        hipLaunchKernelGGL(k_mx_quantise<DT>, dim3(walk_blocks(x.rows, S, sizeof(ElemT<DT>), kAhead<false>)), 256, 0, st,
                           static_cast<const ElemT<DT>*>(x.p), x.rows, K, x.ld, S, codes, scales);
        return hipGetLastError();
    });
}

hipError_t launch_mx_dequantise(const gf_mx_rows& w, const MatOut& out, hipStream_t st) {
    const uint32_t S = mx_chunks(w.K);
    return by_type(out.dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        hipLaunchKernelGGL(k_mx_dequantise<DT>, dim3(walk_blocks(w.rows, S, sizeof(ElemT<DT>), kAhead<true>)), 256, 0, st, w, S,
                           static_cast<ElemT<DT>*>(out.p), out.ld);
        return hipGetLastError();
    });
}

}  // namespace gf
