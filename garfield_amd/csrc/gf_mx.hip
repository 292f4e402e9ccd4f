// Rows in microscaled 4-bit floating point: quantisation, products, gradient
// (gfx950, wave64).  The format and its layout are described at gf_mx_rows.
#include "gf_mx_device.h"

namespace gf {
namespace {

__device__ __forceinline__ float code_value(uint32_t c) {
    const uint32_t m = c & 7u;
    const float v = m < 2u ? 0.5f * float(m) : __uint_as_float(((m >> 1) + 126u) << 23 | (m & 1u) << 22);
    return c & 8u ? -v : v;
}
__device__ __forceinline__ uint32_t code_of(float v) {
    const float a = fabsf(v);
    const uint32_t c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
    return c | (__float_as_uint(v) >> 31) << 3;
}
// The scale byte of a block whose magnitudes' largest bit pattern is top:
// floor(log2) is the exponent field - 127 (subnormals fall to byte 0 anyway),
// 2 less for the grid's largest binade.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
    const uint32_t e = top >> 23;
    return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}

// One thread a block of 32 values.
template <int DT>
__global__ __launch_bounds__(256) void k_mx_quantise(const ElemT<DT>* x, uint64_t rows, uint32_t K,
                                                     uint64_t ld, uint32_t nb, uint8_t* codes, uint8_t* scales) {
    const uint64_t i = uint64_t(blockIdx.x) * 256u + threadIdx.x;
    if (i >= rows * nb) return;
    const uint64_t r = i / nb;
    const uint32_t k0 = uint32_t(i % nb) * 32u;
    float v[32];
    uint32_t top = 0;
    for (uint32_t j = 0; j < 32u; ++j) {
        v[j] = k0 + j < K ? float(x[r * ld + k0 + j]) : 0.0f;
        top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    }
    const uint32_t byte = scale_byte(top);
    const float inv = __uint_as_float((254u - min(byte, 253u)) << 23);
    uint32_t w[4];
    for (uint32_t q = 0; q < 4u; ++q) {
        w[q] = 0;
        for (uint32_t j = 0; j < 8u; ++j)
            if (byte != 255u) w[q] |= code_of(v[q * 8u + j] * inv) << (4u * j);
    }
    reinterpret_cast<uint4*>(codes)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    scales[i] = uint8_t(byte);
}

template <int DT>
__global__ __launch_bounds__(256) void k_mx_dequantise(gf_mx_rows w, uint32_t nb, ElemT<DT>* out, uint64_t ld) {
    const uint64_t i = uint64_t(blockIdx.x) * 256u + threadIdx.x;
    if (i >= w.rows * nb) return;
    const uint64_t r = i / nb;
    const uint32_t k0 = uint32_t(i % nb) * 32u;
    const float s = mx_scale(w.scales[i]);
    for (uint32_t j = 0; j < 32u && k0 + j < w.K; ++j)
        out[r * ld + k0 + j] = ElemT<DT>(code_value(w.codes[i * 16u + j / 2u] >> (j % 2u * 4u) & 15u) * s);
}

// Element k of row r.
struct FromRows {
    gf_mx_rows w;
    uint32_t nb;
    __device__ __forceinline__ float operator()(uint64_t r, uint32_t k) const {
        const uint64_t b = r * nb + k / 32u;
        return code_value(w.codes[b * 16u + k % 32u / 2u] >> (k % 2u * 4u) & 15u) * mx_scale(w.scales[b]);
    }
};
template <int DT>
struct FromMatrix {
    const ElemT<DT>* p;
    uint64_t ld;
    __device__ __forceinline__ float operator()(uint64_t r, uint32_t k) const { return float(p[r * ld + k]); }
};

// out[m][n] = sum over j < J of A(m, j) * B, B = w(n, j), or w(j, n) with TR.
template <class A, int OT, bool TR>
__global__ __launch_bounds__(256) void k_mx_product(A a, FromRows w, uint32_t M, uint32_t N, uint32_t J,
                                                    ElemT<OT>* out, uint64_t ldo) {
    __shared__ float sa[16][17], sb[16][17];
    const uint32_t tx = threadIdx.x & 15u, ty = threadIdx.x >> 4;
    const uint64_t m0 = uint64_t(blockIdx.y) * 16u, n0 = uint64_t(blockIdx.x) * 16u;
    float acc = 0.0f;
    for (uint32_t j0 = 0; j0 < J; j0 += 16u) {
        sa[ty][tx] = m0 + ty < M && j0 + tx < J ? a(m0 + ty, j0 + tx) : 0.0f;
        if (TR)
            sb[tx][ty] = n0 + tx < N && j0 + ty < J ? w(j0 + ty, uint32_t(n0) + tx) : 0.0f;
        else
            sb[ty][tx] = n0 + ty < N && j0 + tx < J ? w(n0 + ty, j0 + tx) : 0.0f;
        __syncthreads();
        for (uint32_t j = 0; j < 16u; ++j) acc = fmaf(sa[ty][j], sb[tx][j], acc);
        __syncthreads();
    }
    if (m0 + ty < M && n0 + tx < N) out[(m0 + ty) * ldo + n0 + tx] = ElemT<OT>(acc);
}

template <bool TR, class A>
hipError_t product(A a, const gf_mx_rows& w, uint32_t M, uint32_t N, uint32_t J, const MatOut& out, hipStream_t st) {
    return by_type(out.dtype, [&](auto ot) {
        constexpr int OT = decltype(ot)::value;
        hipLaunchKernelGGL((k_mx_product<A, OT, TR>), dim3((N + 15u) / 16u, (M + 15u) / 16u), 256, 0, st, a,
                           FromRows{w, 4u * mx_chunks(w.K)}, M, N, J, static_cast<ElemT<OT>*>(out.p), out.ld);
        return hipGetLastError();
    });
}

}  // namespace

hipError_t launch_mx_quantise(const MatIn& x, uint32_t K, uint8_t* codes, uint8_t* scales, hipStream_t st) {
    const uint32_t nb = 4u * mx_chunks(K);
    return by_type(x.dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        hipLaunchKernelGGL(k_mx_quantise<DT>, dim3(uint32_t((x.rows * nb + 255u) / 256u)), 256, 0, st,
                           static_cast<const ElemT<DT>*>(x.p), x.rows, K, x.ld, nb, codes, scales);
        return hipGetLastError();
    });
}

hipError_t launch_mx_dequantise(const gf_mx_rows& w, const MatOut& out, hipStream_t st) {
    const uint32_t nb = 4u * mx_chunks(w.K);
    return by_type(out.dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        hipLaunchKernelGGL(k_mx_dequantise<DT>, dim3(uint32_t((w.rows * nb + 255u) / 256u)), 256, 0, st, w, nb,
                           static_cast<ElemT<DT>*>(out.p), out.ld);
        return hipGetLastError();
    });
}

hipError_t launch_mx_product(const MatIn& x, const gf_mx_rows& w, const MatOut& out, void*, hipStream_t st) {
    return by_type(x.dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        return product<false>(FromMatrix<DT>{static_cast<const ElemT<DT>*>(x.p), x.ld}, w, uint32_t(x.rows),
                              uint32_t(w.rows), w.K, out, st);
    });
}

hipError_t launch_mx_product_grad(const MatIn& dy, const gf_mx_rows& w, const MatOut& dx, void*, hipStream_t st) {
    return by_type(dy.dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        return product<true>(FromMatrix<DT>{static_cast<const ElemT<DT>*>(dy.p), dy.ld}, w,
                             uint32_t(dy.rows), w.K, uint32_t(w.rows), dx, st);
    });
}

size_t mx_workspace(int32_t, int32_t, uint64_t, uint64_t, uint32_t) { return 0; }

}  // namespace gf
