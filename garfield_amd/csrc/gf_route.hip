// Routing of queries (tokens) to cells (experts) and its gradient (gfx950,
// wave64).  The definition is at gf_route in the header.
//
// Both are small passes over T x E logits.  Sixteen lanes hold a row, so a wave
// works on four; all they exchange goes through data-parallel moves within
// their sixteen lanes or a few words of LDS of their own wave, and no barrier
// stands between the load of a row and its result.
//
// Which entries are chosen must not hang on the last bit of a 32-bit
// exponential.  Keys (score + bias) are computed in 32 bits with a bound on
// their error; a row in which a comparison that the result hangs on is closer
// than that bound is done again, by the whole wave, with keys in 64 bits.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "gf_operators.h"

namespace gf {
namespace {

constexpr float kLargest = 3.4028234663852886e38f;
constexpr float kNone = -__builtin_huge_valf();
constexpr uint32_t kRowsPerWave = 4;

// ---- sixteen lanes -----------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __uint_as_float(uint32_t(__builtin_amdgcn_mov_dpp(int(__float_as_uint(v)), CTRL, 0xF, 0xF, true)));
}
// Over the sixteen lanes, the same in all of them (rotations by 8, 4, 2, 1).
__device__ __forceinline__ float max16(float v) {
    v = fmaxf(v, dpp<0x128>(v));
    v = fmaxf(v, dpp<0x124>(v));
    v = fmaxf(v, dpp<0x122>(v));
    return fmaxf(v, dpp<0x121>(v));
}
__device__ __forceinline__ float sum16(float v) {
    v += dpp<0x128>(v);
    v += dpp<0x124>(v);
    v += dpp<0x122>(v);
    return v + dpp<0x121>(v);
}
// The lanes of the sixteen for which p holds, as bits 0 to 15.
__device__ __forceinline__ uint32_t ballot16(bool p) {
    return uint32_t(__ballot(p) >> (threadIdx.x & 48u)) & 0xFFFFu;
}
// Orders a wave's own LDS accesses.
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ---- rows --------------------------------------------------------------------
template <class T>
struct __attribute__((packed, aligned(1))) Vec16 {
    T v[16 / sizeof(T)];
};
// Entries first .. first + V - 1 of a row of E, first = V times the lane of
// sixteen, -inf beyond its end: in 16-byte pieces where the lanes share the row
// evenly, else by way of 16 V words of LDS.
template <int V, class T>
__device__ __forceinline__ void load_row(const T* row, uint32_t first, uint32_t E, float* staged, float* l) {
    constexpr int W = 16 / sizeof(T);
    if (V >= W && E == 16u * V) {
#pragma unroll
        for (int c = 0; c < V; c += W) {
            const Vec16<T> q = *reinterpret_cast<const Vec16<T>*>(row + first + c);
#pragma unroll
            for (int j = 0; j < W && c + j < V; ++j) l[c + j] = float(q.v[j]);
        }
    } else {
#pragma unroll 4
        for (uint32_t e = threadIdx.x & 15u; e < 16u * V; e += 16u) staged[e] = e < E ? float(row[e]) : kNone;
        wave_lds_sync();
#pragma unroll
        for (int j = 0; j < V; ++j) l[j] = staged[first + j];
        wave_lds_sync();
    }
}
// A masked entry (-inf or NaN, in the logit or the bias) as -inf, +inf as the
// largest finite value.
__device__ __forceinline__ float entry(float l, const float* bias, uint32_t e) {
    if (!(l > kNone) || (bias && !(bias[e] > kNone))) return kNone;
    return fminf(l, kLargest);
}

// exp to 2^-17 of itself or better, below 2^-126 0.
__device__ __forceinline__ float exp_near(float v) { return __builtin_amdgcn_exp2f(v * 1.4426950408889634f); }
__device__ __forceinline__ float sigmoid(float v) { return 1.0f / (1.0f + expf(-v)); }

// ---- one row by the whole wave, keys in 64 bits --------------------------------
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
    const uint64_t u = uint64_t(__double_as_longlong(v));
    const uint32_t lo = uint32_t(__builtin_amdgcn_mov_dpp(int(uint32_t(u)), CTRL, 0xF, 0xF, true));
    const uint32_t hi = uint32_t(__builtin_amdgcn_mov_dpp(int(uint32_t(u >> 32)), CTRL, 0xF, 0xF, true));
    return __longlong_as_double((long long)(uint64_t(hi) << 32 | lo));
}
__device__ __forceinline__ double lane64(double v, int lane) {
    const uint64_t u = uint64_t(__double_as_longlong(v));
    const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(u)), lane));
    const uint32_t hi = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(u >> 32)), lane));
    return __longlong_as_double((long long)(uint64_t(hi) << 32 | lo));
}
// f over the wave: within sixteen lanes by rotations, then the four sixteens.
template <class F>
__device__ __forceinline__ double wave_fold(double v, F f) {
    v = f(v, dpp64<0x128>(v));
    v = f(v, dpp64<0x124>(v));
    v = f(v, dpp64<0x122>(v));
    v = f(v, dpp64<0x121>(v));
    return f(f(lane64(v, 0), lane64(v, 16)), f(lane64(v, 32), lane64(v, 48)));
}
__device__ __forceinline__ double wave_max(double v) {
    return wave_fold(v, [](double a, double b) { return fmax(a, b); });
}
__device__ __forceinline__ double wave_sum(double v) {
    return wave_fold(v, [](double a, double b) { return a + b; });
}
// The largest, then the one of the lowest index.
__device__ __forceinline__ void better(double& v, uint32_t& i, double u, uint32_t j) {
    if (u > v || (u == v && j < i)) v = u, i = j;
}
template <int CTRL>
__device__ __forceinline__ void better_dpp(double& v, uint32_t& i) {
    better(v, i, dpp64<CTRL>(v), uint32_t(__builtin_amdgcn_mov_dpp(int(i), CTRL, 0xF, 0xF, true)));
}
__device__ __forceinline__ void wave_best(double& v, uint32_t& i) {
    better_dpp<0x128>(v, i);
    better_dpp<0x124>(v, i);
    better_dpp<0x122>(v, i);
    better_dpp<0x121>(v, i);
    double w = lane64(v, 0);
    uint32_t j = uint32_t(__builtin_amdgcn_readlane(int(i), 0));
#pragma unroll
    for (int l = 16; l < 64; l += 16) better(w, j, lane64(v, l), uint32_t(__builtin_amdgcn_readlane(int(i), l)));
    v = w, i = j;
}
// key: E doubles of LDS of this wave.
template <class T>
__device__ __attribute__((noinline)) void choose_exact(const gf_route_opts& o, const T* row, uint32_t E, const float* bias,
                                                       double* key, int32_t* chosen) {
    const uint32_t lane = threadIdx.x & 63u;
    double mx = kNone, z = 0.0;
    for (uint32_t e = lane; e < E; e += 64u) mx = fmax(mx, double(entry(float(row[e]), bias, e)));
    mx = wave_max(mx);
    for (uint32_t e = lane; e < E; e += 64u) {
        const float l = entry(float(row[e]), bias, e);
        const double x = exp(o.score == GF_SCORE_SIGMOID ? -double(l) : double(l) - mx);
        key[e] = l > kNone ? x : -1.0;   // a lane reads only what it wrote
        z += l > kNone ? x : 0.0;
    }
    z = wave_sum(z);
    for (uint32_t e = lane; e < E; e += 64u) {
        const double x = key[e], s = o.score == GF_SCORE_SIGMOID ? 1.0 / (1.0 + x) : x / z;
        key[e] = x < 0.0 ? double(kNone) : s + (bias ? double(bias[e]) : 0.0);
    }
    wave_lds_sync();
    if (o.groups > 1u) {
        const uint32_t gs = E / o.groups;
        double rank = kNone;
        if (lane < o.groups) {
            double best = kNone, second = kNone;
#pragma unroll 4
            for (uint32_t e = lane * gs; e < (lane + 1u) * gs; ++e) {
                second = fmax(second, fmin(best, key[e]));
                best = fmax(best, key[e]);
            }
            rank = best + (o.group_score == GF_GROUP_TOP2 && second > kNone ? second : 0.0);
        }
        bool kept = lane >= o.groups;
        for (uint32_t r = 0; r < o.keep_groups; ++r) {
            double v = kept ? double(kNone) : rank;
            uint32_t i = kept ? ~0u : lane;
            wave_best(v, i);
            kept |= i == lane;
        }
        wave_lds_sync();
        if (!kept)
            for (uint32_t e = lane * gs; e < (lane + 1u) * gs; ++e) key[e] = kNone;
        wave_lds_sync();
    }
    for (uint32_t r = 0; r < o.k; ++r) {
        double v = kNone;
        uint32_t i = ~0u;
        for (uint32_t e = lane; e < E; e += 64u)
            if (key[e] > v) v = key[e], i = e;
        wave_best(v, i);
        if (lane == 0) {
            chosen[r] = int32_t(i);   // ~0: none left
            if (i < E) key[i] = kNone;
        }
        wave_lds_sync();
    }
}

// Dynamic LDS of k_route in words: the block's load counters; per wave the
// chosen ids and the rows' keys and group ranks, or one row's keys in 64 bits.
template <int V, uint32_t WAVES>
struct RouteLds {
    static constexpr uint32_t kKeys = 16u * V, kRow = kKeys + GF_ROUTE_MAX_GROUPS;
    static constexpr uint32_t kWave = kRowsPerWave * (GF_ROUTE_MAX_K + kRow);
    static constexpr uint32_t kBytes = 4u * (kKeys + WAVES * kWave);
};

// The three best of a lane's keys, the lower index first among equals (keys
// are added by ascending index).
struct Three {
    float v[3];
    uint32_t i[3];
    __device__ __forceinline__ void clear() { v[0] = v[1] = v[2] = kNone, i[0] = i[1] = i[2] = 0; }
    __device__ __forceinline__ void add(float k, uint32_t at) {
        const bool a = k > v[0], b = k > v[1], c = k > v[2];
        i[2] = b ? i[1] : c ? at : i[2];
        i[1] = a ? i[0] : b ? at : i[1];
        i[0] = a ? at : i[0];
        v[2] = __builtin_amdgcn_fmed3f(k, v[1], v[2]);
        v[1] = __builtin_amdgcn_fmed3f(k, v[0], v[1]);
        v[0] = fmaxf(v[0], k);
    }
};

// A lane holds V consecutive entries of its row: the lowest lane that has the
// largest key has the lowest index too.  It keeps its three best at hand and
// looks through its V again only when all are chosen and it had more: with
// k = 8 that is once in four rows.  Groups that are whole lanes are ranked from the lanes' two
// best, by moves between lanes; others through LDS.
template <class T, int V, uint32_t WAVES>
__global__ __launch_bounds__(64 * WAVES, V >= 32 ? 2 : 4) void k_route(gf_route_opts o, const T* logits, uint32_t rows,
                                                                       uint32_t E, uint64_t ld, const float* bias,
                                                                       int32_t* ids, float* weights, int32_t* load) {
    extern __shared__ __align__(16) uint32_t lds[];
    const uint32_t lane = threadIdx.x & 63u, c = lane & 15u, mine = lane >> 4, wave = threadIdx.x >> 6;
    const uint32_t first = c * V;
    using L = RouteLds<V, WAVES>;
    uint32_t* count = lds;
    uint32_t* own = lds + L::kKeys + wave * L::kWave;
    int32_t* chosen = reinterpret_cast<int32_t*>(own) + mine * GF_ROUTE_MAX_K;
    float* keys = reinterpret_cast<float*>(own + kRowsPerWave * GF_ROUTE_MAX_K);
    float *mykeys = keys + mine * L::kRow, *myranks = mykeys + L::kKeys;
    if (load) {
        for (uint32_t e = threadIdx.x; e < E; e += 64u * WAVES) count[e] = 0;
        __syncthreads();
    }
    const bool by_score = bias || (o.groups > 1u && o.group_score == GF_GROUP_TOP2);
    const bool soft = o.score == GF_SCORE_SOFTMAX;
    // groups of whole lanes, `span` each
    const bool whole = o.groups > 1u && E == 16u * V && 16u % o.groups == 0;
    const uint32_t span = whole ? 16u / o.groups : 1u;
    const uint32_t gs = E / o.groups, magic = ((1u << 20) + gs - 1u) / gs;   // e / gs = e magic >> 20 below 1024

    for (uint64_t t0 = (uint64_t(blockIdx.x) * WAVES + wave) * kRowsPerWave; t0 < rows;
         t0 += uint64_t(gridDim.x) * WAVES * kRowsPerWave) {
        const bool row_ok = t0 + mine < rows;
        const uint64_t t = row_ok ? t0 + mine : rows - 1u;   // lanes without a row repeat the last, unstored
        const T* row = logits + t * ld;
        float key[V];
        load_row<V>(row, first, E, mykeys, key);
        float mx = kNone, top = 0.0f;   // top: the largest |bias|
        if (bias) {
            float b[V];
            load_row<V>(bias, first, E, mykeys, b);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                key[j] = b[j] > kNone ? key[j] : kNone;
                top = fmaxf(top, b[j] > kNone ? fabsf(b[j]) : 0.0f);
            }
            top = max16(top);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {   // fmaxf takes a NaN for -inf
            key[j] = fminf(fmaxf(key[j], kNone), kLargest);
            mx = fmaxf(mx, key[j]);
        }
        mx = max16(mx);
        const float lift = mx > kNone ? mx : 0.0f;
        float z = 1.0f;   // of the softmax over the row
        if (soft && (by_score || !o.renormalise)) {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float e = exp_near(key[j] - lift);   // 0 for a masked entry
                sum += e;
                if (by_score) key[j] = key[j] > kNone ? e : -1.0f;
            }
            z = sum16(sum);
        }
        // How far a 32-bit key k may be off: rel (|k| + top) + least.  Softmax: the
        // difference and its product with log2 e are rounded (|difference| below
        // 104 where the result is not 0: 2^-16 in all), and a sum of E terms is
        // off by (V + 4) 2^-24 of itself.  Sigmoid: the error of the exponential
        // e weighs e / (1 + e)^2 times its argument, below 1/4; the rest is a few
        // units in the last place.
        const float rel = soft ? 0x1p-15f : 0x1p-21f, least = soft ? 0x1p-126f : 0x1p-24f;
        if (by_score) {
            const float inv = 1.0f / z;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (soft)
                    key[j] = key[j] < 0.0f ? kNone : key[j] * inv;
                else
                    key[j] = key[j] > kNone ? __builtin_amdgcn_rcpf(1.0f + exp_near(-key[j])) : kNone;
            }
            if (bias) {
                float b[V];
                load_row<V>(bias, first, E, mykeys, b);
#pragma unroll
                for (int j = 0; j < V; ++j) key[j] = key[j] > kNone ? key[j] + b[j] : kNone;
            }
        }
        auto off = [&](float k) { return rel * (fabsf(k) + top) + least; };
        bool close = false;   // a comparison that 32 bits do not decide
        Three best;
        best.clear();
        auto rank_of = [&](float first_best, float second_best) {
            return first_best + (o.group_score == GF_GROUP_TOP2 && second_best > kNone ? second_best : 0.0f);
        };
        // a rank is the sum of two keys at most; no key is below -top, so neither
        // is beyond |rank| + top
        auto too_close = [&](float low, float high) {
            return by_score && high > kNone && low - high <= 2.0f * (off(low) + off(high) + 2.0f * rel * top);
        };
        if (o.groups == 1u || whole) {
#pragma unroll
            for (int j = 0; j < V; ++j) best.add(key[j], first + j);
            if (whole) {
                float u = best.v[0], d = best.v[1];
                for (uint32_t s = 1; s < span; s <<= 1) {
                    const float u2 = __shfl_xor(u, int(s)), d2 = __shfl_xor(d, int(s));
                    d = fmaxf(fmaxf(d, d2), fminf(u, u2));
                    u = fmaxf(u, u2);
                }
                const float rank = rank_of(u, d);
                // of the fifteen other lanes, those of a better group (each group
                // `span` times; the own one never)
                uint32_t ahead = 0;
                float turn = rank;
#pragma unroll
                for (uint32_t n = 1; n < 16u; ++n) {
                    turn = dpp<0x121>(turn);   // lane c has lane c - n's (of sixteen)
                    ahead += turn > rank || (turn == rank && (c - n & 15u) / span < c / span);
                }
                const bool kept = ahead < o.keep_groups * span;
                close = too_close(-max16(kept ? -rank : kNone), max16(kept ? kNone : rank));
                if (!kept) best.clear();
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) mykeys[first + j] = key[j];
            wave_lds_sync();
            // `share` lanes a group where there are fewer than sixteen groups, or
            // up to four groups a lane; lanes start at different places of their
            // groups, in different banks
            const uint32_t share = o.groups <= 2u ? 8u : o.groups <= 4u ? 4u : o.groups <= 8u ? 2u : 1u;
            for (uint32_t i = 0; i * (16u / share) < o.groups; ++i) {
                const uint32_t g = i * (16u / share) + c / share, p = c % share;
                float u = kNone, d = kNone;
                if (g < o.groups && p < gs) {
                    const uint32_t n = (gs - p + share - 1u) / share;   // entries p, p + share, ..
                    uint32_t at = c % n;
#pragma unroll 4
                    for (uint32_t e = 0; e < n; ++e) {
                        const float v = mykeys[g * gs + p + at * share];
                        at = at + 1u == n ? 0u : at + 1u;
                        d = __builtin_amdgcn_fmed3f(v, u, d);
                        u = fmaxf(u, v);
                    }
                }
                for (uint32_t s = 1; s < share; s <<= 1) {
                    const float u2 = __shfl_xor(u, int(s)), d2 = __shfl_xor(d, int(s));
                    d = fmaxf(fmaxf(d, d2), fminf(u, u2));
                    u = fmaxf(u, u2);
                }
                if (p == 0 && g < o.groups) myranks[g] = rank_of(u, d);
            }
            wave_lds_sync();
            // a group's place among the ranks; kept are the first keep_groups
            uint64_t kept = 0;
            float low = -kNone, high = kNone;   // the last kept rank, the first not kept
            for (uint32_t i = 0; i < o.groups; i += 16u) {
                const uint32_t g = i + c;
                const float v = g < o.groups ? myranks[g] : kNone;
                uint32_t place = 0;
#pragma unroll 4
                for (uint32_t n = 0; n < o.groups; ++n) {
                    const float u = myranks[n];
                    place += u > v || (u == v && n < g);
                }
                const bool in = g < o.groups && place < o.keep_groups;
                kept |= uint64_t(ballot16(in)) << i;
                if (in) low = fminf(low, v);
                else if (g < o.groups) high = fmaxf(high, v);
            }
            close = too_close(-max16(-low), max16(high));
            // the entries' groups, counted up; not ahead of the loop over rows, which
            // would take a register each
            uint32_t g = first * magic >> 20, left = (g + 1u) * gs - first;
            asm volatile("" : "+v"(g), "+v"(left));
#pragma unroll
            for (int j = 0; j < V; ++j) {
                key[j] = kept >> (g & 63u) & 1u ? key[j] : kNone;
                const bool over = --left == 0;
                g += over, left = over ? gs : left;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) best.add(key[j], first + j);
        }
        float before = 0.0f;
        bool more = best.v[2] > kNone;   // the lane may have a fourth
        for (uint32_t n = 0; n <= o.k; ++n) {
            const float m = max16(best.v[0]);
            if (by_score && n && m > kNone) close |= before - m <= off(before) + off(m);
            before = m;
            if (n == o.k) break;
            const uint32_t who = ballot16(best.v[0] == m && m > kNone);
            if (!who && c == 0) chosen[n] = -1;
            if (who && c == uint32_t(__ffs(int(who))) - 1u) {
                const uint32_t last = best.i[0];
                chosen[n] = int32_t(last);
                best.v[0] = best.v[1], best.i[0] = best.i[1];
                best.v[1] = best.v[2], best.i[1] = best.i[2];
                best.v[2] = kNone;
                if (V > 3 && more && !(best.v[0] > kNone)) {   // look again, behind (m, last)
                    best.clear();
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        best.add(key[j] < m || (key[j] == m && first + j > last) ? key[j] : kNone, first + j);
                    more = best.v[2] > kNone;
                }
            }
        }
        wave_lds_sync();
        if (by_score) {
            uint64_t again = __ballot(close && c == 0);
            while (again) {
                const uint32_t r = uint32_t(__ffsll((long long)again) - 1) / 16u;
                again &= again - 1u;
                choose_exact(o, logits + min(t0 + r, uint64_t(rows) - 1u) * ld, E, bias, reinterpret_cast<double*>(keys),
                             reinterpret_cast<int32_t*>(own) + r * GF_ROUTE_MAX_K);
            }
        }
        // up to four of the row's choices a lane
        float s[4], l[4], sum = 0.0f, peak = kNone;
        int32_t id[4];
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const uint32_t n = i * 16u + c;
            id[i] = n < o.k ? chosen[n] : -1;
            l[i] = id[i] >= 0 ? fminf(float(row[id[i]]), kLargest) : kNone;
            peak = fmaxf(peak, l[i]);
        }
        if (o.renormalise) mx = max16(peak);   // the softmax over the row cancels
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            s[i] = id[i] < 0 ? 0.0f : soft ? expf(l[i] - mx) / (o.renormalise ? 1.0f : z) : sigmoid(l[i]);
            sum += s[i];
        }
        if (o.renormalise) sum = sum16(sum);
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const uint32_t n = i * 16u + c;
            if (!row_ok || n >= o.k) continue;
            ids[t * o.k + n] = id[i];
            weights[t * o.k + n] = o.scale * (o.renormalise ? sum > 0.0f ? s[i] / sum : 0.0f : s[i]);
            if (load && id[i] >= 0) atomicAdd(count + id[i], 1u);
        }
        wave_lds_sync();
    }
    if (load) {   // whole numbers: the order does not matter
        __syncthreads();
        for (uint32_t e = threadIdx.x; e < E; e += 64u * WAVES)
            if (count[e]) atomicAdd(load + e, int32_t(count[e]));
    }
}

__global__ void k_route_clear(int32_t* load, uint32_t E) {
    const uint32_t e = blockIdx.x * 256u + threadIdx.x;
    if (e < E) load[e] = 0;
}

// The gradient, sixteen lanes a row as above: the k chosen entries' terms are
// put into a row of LDS that is written out whole; the softmax over all
// entries adds its term to every live one.
constexpr uint32_t kGradWaves = 4;
template <class T>
__global__ __launch_bounds__(64 * kGradWaves) void k_route_grad(gf_route_opts o, const T* logits, uint32_t rows, uint32_t E,
                                                            uint64_t ld, const float* bias, const int32_t* ids,
                                                            const float* dweights, T* dlogits, uint64_t ldd) {
    extern __shared__ __align__(16) uint32_t lds[];
    const uint32_t lane = threadIdx.x & 63u, c = lane & 15u, wave = threadIdx.x >> 6;
    const uint32_t pitch = E + 7u & ~7u;
    float* d = reinterpret_cast<float*>(lds) + (wave * kRowsPerWave + (lane >> 4)) * pitch;
    const bool soft = o.score == GF_SCORE_SOFTMAX;
    for (uint64_t t0 = (uint64_t(blockIdx.x) * kGradWaves + wave) * kRowsPerWave; t0 < rows;
         t0 += uint64_t(gridDim.x) * kGradWaves * kRowsPerWave) {
        const bool row_ok = t0 + (lane >> 4) < rows;
        const uint64_t t = row_ok ? t0 + (lane >> 4) : rows - 1u;
        const T* row = logits + t * ld;
        for (uint32_t e = c * 4u; e < pitch; e += 64u) *reinterpret_cast<float4*>(d + e) = make_float4(0, 0, 0, 0);
        float l[4], g[4], s[4], sum = 0.0f, peak = kNone, mx = kNone, z = 0.0f;
        int32_t id[4];
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const uint32_t n = i * 16u + c;
            id[i] = n < o.k ? ids[t * o.k + n] : -1;
            if (id[i] < 0 || uint32_t(id[i]) >= E) id[i] = -1;
            l[i] = id[i] >= 0 ? entry(float(row[id[i]]), bias, uint32_t(id[i])) : kNone;
            if (!(l[i] > kNone)) id[i] = -1;
            g[i] = id[i] >= 0 ? dweights[t * o.k + n] : 0.0f;
            peak = fmaxf(peak, l[i]);
        }
        const bool all = soft && !o.renormalise;
        if (all) {
            for (uint32_t e = c; e < E; e += 16u) mx = fmaxf(mx, entry(float(row[e]), bias, e));
            mx = max16(mx);
            for (uint32_t e = c; e < E; e += 16u) {
                const float v = entry(float(row[e]), bias, e);
                if (v > kNone) z += expf(v - mx);
            }
            z = sum16(z);
        } else {
            mx = max16(peak), z = 1.0f;
        }
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            s[i] = id[i] < 0 ? 0.0f : soft ? expf(l[i] - mx) / z : sigmoid(l[i]);
            sum += s[i];
        }
        float mean = 0.0f;
        if (o.renormalise) {
            sum = sum16(sum);
            const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
            float share[4];
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) share[i] = s[i] * inv, mean += g[i] * share[i];
            mean = sum16(mean);
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) g[i] = o.scale * (g[i] - mean) * share[i] * (soft ? 1.0f : 1.0f - s[i]);
        } else if (soft) {
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) mean += g[i] * s[i];
            mean = sum16(mean);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) g[i] *= o.scale * s[i] * (1.0f - s[i]);
        }
        wave_lds_sync();
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i)
            if (id[i] >= 0) d[id[i]] = g[i];
        wave_lds_sync();
        if (all) {
            for (uint32_t e = c; e < E; e += 16u) {
                const float v = entry(float(row[e]), bias, e);
                d[e] = v > kNone ? o.scale * (expf(v - mx) / z) * (d[e] - mean) : 0.0f;
            }
            wave_lds_sync();
        }
        if (row_ok) {
            constexpr uint32_t W = 16 / sizeof(T);
            T* out = dlogits + t * ldd;
            for (uint32_t e = c * W; e < E; e += 16u * W) {
                Vec16<T> q;
#pragma unroll
                for (uint32_t j = 0; j < W; ++j) q.v[j] = T(d[e + j]);   // pitch covers the tail
                if (e + W <= E)
                    *reinterpret_cast<Vec16<T>*>(out + e) = q;
                else
                    for (uint32_t j = 0; e + j < E; ++j) out[e + j] = T(d[e + j]);
            }
        }
        wave_lds_sync();
    }
}

template <class F>
hipError_t by_type(int32_t dtype, F&& f) {
    if (dtype == GF_F32) return f(float());
    if (dtype == GF_F16) return f(_Float16());
    return f(__bf16());
}
template <class F>
hipError_t by_width(uint32_t E, F&& f) {
    if (E <= 16u) return f(std::integral_constant<int, 1>());
    if (E <= 32u) return f(std::integral_constant<int, 2>());
    if (E <= 64u) return f(std::integral_constant<int, 4>());
    if (E <= 128u) return f(std::integral_constant<int, 8>());
    if (E <= 256u) return f(std::integral_constant<int, 16>());
    if (E <= 512u) return f(std::integral_constant<int, 32>());
    return f(std::integral_constant<int, 64>());
}
// A wave has four rows at a time; beyond this many blocks it takes more.
uint32_t route_blocks(uint64_t rows, uint32_t waves) {
    return uint32_t(std::min<uint64_t>((rows + waves * kRowsPerWave - 1u) / (waves * kRowsPerWave), 8192u / waves));
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
        return by_width(E, [&](auto width) {
            using T = decltype(v);
            constexpr int V = decltype(width)::value;
            auto go = [&](auto waves) {
                constexpr uint32_t W = decltype(waves)::value;
                constexpr uint32_t kLds = RouteLds<V, W>::kBytes;
                hipLaunchKernelGGL((k_route<T, V, W>), dim3(route_blocks(logits.rows, W)), 64 * W, kLds, st, o,
                                   static_cast<const T*>(logits.p), uint32_t(logits.rows), E, logits.ld, bias, ids, weights,
                                   load);
                return hipGetLastError();
            };
            // a block ends with an atomic addition for every entry that it counted:
            // where rows fill the chip anyway, few large blocks
            if constexpr (V <= 16)
                if (load && logits.rows >= 8192u) return go(std::integral_constant<uint32_t, 16>());
            return go(std::integral_constant<uint32_t, 4>());
        });
    });
}

hipError_t launch_route_grad(const gf_route_opts& o, const MatIn& logits, uint32_t E, const float* bias,
                             const int32_t* ids, const float* dweights, const MatOut& dlogits, hipStream_t st) {
    return by_type(logits.dtype, [&](auto v) {
        using T = decltype(v);
        hipLaunchKernelGGL(k_route_grad<T>, dim3(route_blocks(logits.rows, kGradWaves)), 64 * kGradWaves,
                           kGradWaves * kRowsPerWave * (E + 7u & ~7u) * 4u, st, o, static_cast<const T*>(logits.p),
                           uint32_t(logits.rows), E, logits.ld, bias, ids, dweights, static_cast<T*>(dlogits.p), dlogits.ld);
        return hipGetLastError();
    });
}

}  // namespace gf
