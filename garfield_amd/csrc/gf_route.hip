// Routing of queries (tokens) to cells (experts) and its gradient (gfx950,
// wave64).  The definition is at gf_route in the header.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <type_traits>

#include "gf_operators.h"

namespace gf {
namespace {

constexpr float kLargest = 3.4028234663852886e38f;
constexpr float kNone = -__builtin_huge_valf();

template <int DT>
struct Elem {
    using T = std::conditional_t<DT == GF_F32, float, std::conditional_t<DT == GF_F16, _Float16, __bf16>>;
};

template <class T>
__device__ __forceinline__ T wave_max(T v) {
    for (int o = 32; o; o >>= 1) {
        const T u = __shfl_xor(v, o);
        v = u > v ? u : v;
    }
    return v;
}
template <class T>
__device__ __forceinline__ T wave_sum(T v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// The lane-wise best (largest, then lowest index) over the wave.
__device__ __forceinline__ void wave_best(double& v, uint32_t& i) {
    for (int o = 32; o; o >>= 1) {
        const double u = __shfl_xor(v, o);
        const uint32_t j = __shfl_xor(i, o);
        if (u > v || (u == v && j < i)) v = u, i = j;
    }
}

// A row's logits in LDS, masked entries as -inf; returns nothing else.
template <class T>
__device__ __forceinline__ void read_row(const T* row, uint32_t E, const float* bias, float* l) {
    for (uint32_t e = threadIdx.x; e < E; e += 64u) {
        float v = float(row[e]);
        if (!(v > kNone) || (bias && !(bias[e] > kNone))) v = kNone;
        l[e] = fminf(v, kLargest);
    }
    __syncthreads();
}

// One wave a row; keys in 64 bits.
template <class T>
__global__ __launch_bounds__(64) void k_route(gf_route_opts o, const T* logits, uint32_t rows, uint32_t E, uint64_t ld,
                                              const float* bias, int32_t* ids, float* weights, int32_t* load) {
    __shared__ float l[GF_ROUTE_MAX_E];
    __shared__ double key[GF_ROUTE_MAX_E];
    __shared__ int32_t chosen[GF_ROUTE_MAX_K];
    const uint64_t t = blockIdx.x;
    const uint32_t lane = threadIdx.x;
    read_row(logits + t * ld, E, bias, l);
    float mx = kNone;
    for (uint32_t e = lane; e < E; e += 64u) mx = fmaxf(mx, l[e]);
    mx = wave_max(mx);
    double z = 0.0;
    for (uint32_t e = lane; e < E; e += 64u)
        if (l[e] > kNone) z += exp(double(l[e]) - double(mx));
    z = wave_sum(z);
    auto score = [&](uint32_t e) {
        return o.score == GF_SCORE_SIGMOID ? 1.0 / (1.0 + exp(-double(l[e]))) : exp(double(l[e]) - double(mx)) / z;
    };
    const bool by_score = bias || (o.groups > 1 && o.group_score == GF_GROUP_TOP2);
    for (uint32_t e = lane; e < E; e += 64u) {
        const bool live = l[e] > kNone;
        key[e] = !live ? double(kNone) : by_score ? score(e) + (bias ? double(bias[e]) : 0.0) : double(l[e]);
    }
    __syncthreads();
    if (o.groups > 1) {
        const uint32_t gs = E / o.groups;
        double rank = kNone;
        if (lane < o.groups) {
            double best = kNone, second = kNone;
            for (uint32_t e = lane * gs; e < (lane + 1u) * gs; ++e) {
                if (key[e] > best) second = best, best = key[e];
                else if (key[e] > second) second = key[e];
            }
            rank = best + (o.group_score == GF_GROUP_TOP2 && second > kNone ? second : 0.0);
        }
        bool kept = false;
        for (uint32_t r = 0; r < o.keep_groups; ++r) {
            double v = kept || lane >= o.groups ? double(kNone) : rank;
            uint32_t i = kept || lane >= o.groups ? 0x7FFFFFFFu : lane;
            wave_best(v, i);
            kept |= i == lane;
        }
        __syncthreads();
        if (lane < o.groups && !kept)
            for (uint32_t e = lane * gs; e < (lane + 1u) * gs; ++e) key[e] = kNone;
        __syncthreads();
    }
    for (uint32_t r = 0; r < o.k; ++r) {
        double v = kNone;
        uint32_t i = 0x7FFFFFFFu;
        for (uint32_t e = lane; e < E; e += 64u)
            if (key[e] > v) v = key[e], i = e;
        wave_best(v, i);
        if (lane == 0) {
            chosen[r] = i < E ? int32_t(i) : -1;
            if (i < E) key[i] = kNone;
        }
        __syncthreads();
    }
    const int32_t id = lane < o.k ? chosen[lane] : -1;
    float s = 0.0f;
    if (id >= 0) s = float(score(uint32_t(id)));
    if (o.renormalise && o.score == GF_SCORE_SOFTMAX) {
        const float top = wave_max(id >= 0 ? l[id] : kNone);
        s = id >= 0 ? expf(l[id] - top) : 0.0f;
    }
    const float total = wave_sum(s);
    if (o.renormalise) s = total > 0.0f ? s / total : 0.0f;
    if (lane < o.k) {
        ids[t * o.k + lane] = id;
        weights[t * o.k + lane] = s * o.scale;
        if (load && id >= 0) atomicAdd(load + id, 1);
    }
}

__global__ void k_route_clear(int32_t* load, uint32_t E) {
    const uint32_t e = blockIdx.x * 256u + threadIdx.x;
    if (e < E) load[e] = 0;
}

template <class T>
__global__ __launch_bounds__(64) void k_route_grad(gf_route_opts o, const T* logits, uint32_t rows, uint32_t E,
                                                   uint64_t ld, const float* bias, const int32_t* ids,
                                                   const float* dweights, T* dlogits, uint64_t ldd) {
    __shared__ float l[GF_ROUTE_MAX_E], d[GF_ROUTE_MAX_E];
    const uint64_t t = blockIdx.x;
    const uint32_t lane = threadIdx.x;
    read_row(logits + t * ld, E, bias, l);
    float mx = kNone, z = 0.0f;
    for (uint32_t e = lane; e < E; e += 64u) mx = fmaxf(mx, l[e]), d[e] = 0.0f;
    mx = wave_max(mx);
    for (uint32_t e = lane; e < E; e += 64u)
        if (l[e] > kNone) z += expf(l[e] - mx);
    z = wave_sum(z);
    int32_t id = lane < o.k ? ids[t * o.k + lane] : -1;
    if (id < 0 || uint32_t(id) >= E || !(l[id] > kNone)) id = -1;
    const float g = id >= 0 ? dweights[t * o.k + lane] : 0.0f;
    auto sigmoid = [](float v) { return 1.0f / (1.0f + expf(-v)); };
    float s = 0.0f;
    if (o.score == GF_SCORE_SIGMOID) s = id >= 0 ? sigmoid(l[id]) : 0.0f;
    else {
        const float top = o.renormalise ? wave_max(id >= 0 ? l[id] : kNone) : mx;
        s = id >= 0 ? expf(l[id] - top) / (o.renormalise ? 1.0f : z) : 0.0f;
    }
    __syncthreads();
    if (o.renormalise) {
        const float total = wave_sum(s), share = total > 0.0f ? s / total : 0.0f;
        const float ds = o.scale * (g - wave_sum(g * share)) * share;
        if (id >= 0) d[id] = o.score == GF_SCORE_SOFTMAX ? ds : ds * (1.0f - s);
    } else if (o.score == GF_SCORE_SIGMOID) {
        if (id >= 0) d[id] = o.scale * g * s * (1.0f - s);
    } else {
        const float mean = wave_sum(g * s);
        if (id >= 0) d[id] = g;
        __syncthreads();
        for (uint32_t e = lane; e < E; e += 64u)
            d[e] = l[e] > kNone ? o.scale * (expf(l[e] - mx) / z) * (d[e] - mean) : 0.0f;
    }
    __syncthreads();
    for (uint32_t e = lane; e < E; e += 64u) dlogits[t * ldd + e] = T(d[e]);
}

template <class F>
hipError_t by_type(int32_t dtype, F&& f) {
    if (dtype == GF_F32) return f(float());
    if (dtype == GF_F16) return f(_Float16());
    return f(__bf16());
}

}  // namespace

hipError_t launch_route(const gf_route_opts& o, const MatIn& logits, uint32_t E, const float* bias, int32_t* ids,
                        float* weights, int32_t* load, hipStream_t st) {
    if (load) {
        hipLaunchKernelGGL(k_route_clear, dim3((E + 255u) / 256u), 256, 0, st, load, E);
        if (const hipError_t e = hipGetLastError()) return e;
    }
    if (!logits.rows) return hipSuccess;
    return by_type(logits.dtype, [&](auto v) {
        using T = decltype(v);
        hipLaunchKernelGGL(k_route<T>, dim3(uint32_t(logits.rows)), 64, 0, st, o, static_cast<const T*>(logits.p),
                           uint32_t(logits.rows), E, logits.ld, bias, ids, weights, load);
        return hipGetLastError();
    });
}

hipError_t launch_route_grad(const gf_route_opts& o, const MatIn& logits, uint32_t E, const float* bias,
                             const int32_t* ids, const float* dweights, const MatOut& dlogits, hipStream_t st) {
    return by_type(logits.dtype, [&](auto v) {
        using T = decltype(v);
        hipLaunchKernelGGL(k_route_grad<T>, dim3(uint32_t(logits.rows)), 64, 0, st, o, static_cast<const T*>(logits.p),
                           uint32_t(logits.rows), E, logits.ld, bias, ids, dweights, static_cast<T*>(dlogits.p),
                           dlogits.ld);
        return hipGetLastError();
    });
}

}  // namespace gf
