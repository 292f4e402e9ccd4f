// Routing of queries (tokens) to cells (experts) and its gradient (gfx950,
// wave64).  The definition is at gf_route in the header.
//
// Both are small passes over T x E logits.  Sixteen lanes hold a row of up to 256
// entries, so a wave works on four; a longer row takes the whole wave.  All that
// lanes exchange goes through data-parallel moves or a few words of LDS of their
// own wave, and no barrier stands between the load of a row and its result.
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
// The same over the LANES (16 or 64) of a row: two exchanges of sixteens more.
template <class F>
__device__ __forceinline__ float over_wave(float v, F f) {
    const uint32_t u = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const uint32_t w = __float_as_uint(v);
    const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
template <int LANES>
__device__ __forceinline__ float max_row(float v) {
    v = max16(v);
    return LANES == 16 ? v : over_wave(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int LANES>
__device__ __forceinline__ float sum_row(float v) {
    v = sum16(v);
    return LANES == 16 ? v : over_wave(v, [](float a, float b) { return a + b; });
}
// The row's lanes for which p holds, as bits from 0.
template <int LANES>
__device__ __forceinline__ uint64_t ballot_row(bool p) {
    const uint64_t all = __ballot(p);
    return LANES == 64 ? all : all >> (threadIdx.x & 48u) & 0xFFFFu;
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
// Entries first .. first + V - 1 of a row of E, first = V times the lane of the
// row's LANES, -inf beyond its end: in 16-byte pieces where the lanes share the
// row evenly, else one coalesced entry after the other by way of LDS, a lane's V
// at a pitch of V + 4 for V = 16: their 16-byte reads fall into different banks.
template <int V>
constexpr uint32_t kGap = V >= 16 ? 4 : 0;
template <int LANES, int V, class T>
__device__ __forceinline__ void load_row(const T* row, uint32_t first, uint32_t E, float* staged, float* l) {
    constexpr int W = 16 / sizeof(T);
    if (V >= W && E == uint32_t(LANES) * V) {
#pragma unroll
        for (int c = 0; c < V; c += W) {
            const Vec16<T> q = *reinterpret_cast<const Vec16<T>*>(row + first + c);
#pragma unroll
            for (int j = 0; j < W && c + j < V; ++j) l[c + j] = float(q.v[j]);
        }
    } else {
        const uint32_t c = threadIdx.x & (LANES - 1u);
#pragma unroll
        for (int j = 0; j < V; ++j) l[j] = c + LANES * j < E ? float(row[c + LANES * j]) : kNone;
#pragma unroll
        for (int j = 0; j < V; ++j) staged[c + LANES * j + (c + LANES * j) / V * kGap<V>] = l[j];
        wave_lds_sync();
#pragma unroll
        for (int j = 0; j < V; ++j) l[j] = staged[first + first / V * kGap<V> + j];
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
// e^-lift times the sigmoid of v, lift being 0 or, if v is below -17, at least v.
// There the sigmoid is e^v, but for less than 2^-24 of itself; 1 / (1 + e^-v) would
// be 0 from -88.8 on.  Below 2^-1022 it counts as 0: entries at a type's lowest value.
constexpr float kLeastSigmoid = -708.39642f;
__device__ __forceinline__ float sigmoid(float v, float lift = 0.0f) {
    const bool low = v < -17.0f;
    const float e = expf(low ? v - lift : -v);
    return low ? v < kLeastSigmoid ? 0.0f : e : 1.0f / (1.0f + e);
}
// The lift of a row whose largest chosen logit is top, where weights are shares of
// the chosen sigmoids' sum: shares of what need not underflow.
__device__ __forceinline__ float sigmoid_lift(float top) { return top < -17.0f ? top : 0.0f; }

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
// A lane holds entries lane, lane + 64, ..: N of them.  Few rows come here, but a
// launch waits for the last: its loads are in flight together and its keys in
// registers for the choices (322 rows of 832 in bfloat16, whose groups tie now and then, with the
// gradient: 26 us; with keys read from LDS for every choice 102).
// key: E doubles of LDS of this wave, for the groups' ranks.
template <int N, class T>
__device__ __attribute__((noinline)) void choose_exact(gf_route_opts o, const T* row, uint32_t E, const float* bias,
                                                       double* key, int32_t* chosen) {
    const uint32_t lane = threadIdx.x & 63u;
    double mx = kNone, z = 0.0;
#pragma unroll 4
    for (uint32_t e = lane; e < E; e += 64u) {   // a lane reads only what it wrote
        const float l = entry(float(row[e]), bias, e);
        key[e] = l;
        mx = fmax(mx, double(l));
    }
    mx = wave_max(mx);
    const bool sigmoid = o.score == GF_SCORE_SIGMOID;
    const double lift = mx > kNone ? mx : 0.0;
#pragma unroll 1
    for (uint32_t e = lane; e < E; e += 64u) {   // 0 for a masked entry of a softmax
        const double v = key[e], x = exp(sigmoid ? -v : v - lift);
        key[e] = v > kNone ? x : -1.0;
        z += x;
    }
    z = wave_sum(z);
#pragma unroll 1
    for (uint32_t e = lane; e < E; e += 64u) {
        const double x = key[e];
        key[e] = x < 0.0 ? double(kNone) : (sigmoid ? 1.0 / (1.0 + x) : x / z) + (bias ? double(bias[e]) : 0.0);
    }
    double x[N];
#pragma unroll
    for (int n = 0; n < N; ++n) x[n] = lane + 64u * n < E ? key[lane + 64u * n] : double(kNone);
    if (o.groups > 1u) {
        const uint32_t gs = E / o.groups, share = 1u << (31 - __clz(int(64u / o.groups)));   // lanes a group
        const uint32_t g = lane / share, p = lane % share;
        wave_lds_sync();
        double best = kNone, second = kNone;
        if (g < o.groups) {
#pragma unroll 4
            for (uint32_t e = p; e < gs; e += share) {
                const double v = key[g * gs + e];
                second = fmax(second, fmin(best, v));
                best = fmax(best, v);
            }
        }
        for (uint32_t s = 1; s < share; s <<= 1) {
            const double u = __shfl_xor(best, int(s)), d = __shfl_xor(second, int(s));
            second = fmax(fmax(second, d), fmin(best, u));
            best = fmax(best, u);
        }
        const double rank = best + (o.group_score == GF_GROUP_TOP2 && second > kNone ? second : 0.0);
        uint32_t place = 0;   // of the group among the ranks
        for (uint32_t n = 0; n < o.groups; ++n) {
            const double u = lane64(rank, int(n * share));
            place += u > rank || (u == rank && n < g);
        }
        const uint64_t kept = __ballot(p == 0 && g < o.groups && place < o.keep_groups);
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (!(kept >> (min(lane + 64u * n, E - 1u) / gs * share) & 1u)) x[n] = kNone;
        wave_lds_sync();
    }
    for (uint32_t r = 0; r < o.k; ++r) {
        double v = kNone;
        uint32_t i = ~0u;
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (x[n] > v) v = x[n], i = lane + 64u * n;
        wave_best(v, i);
        if (lane == 0) chosen[r] = int32_t(i);   // ~0: none left
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (i == lane + 64u * n) x[n] = kNone;
    }
    wave_lds_sync();
}

// Dynamic LDS of k_route in words: the block's load counters; per wave the
// chosen ids and the rows' keys and group ranks, or one row's keys in 64 bits.
template <int LANES, int V>
struct RouteLds {
    static constexpr uint32_t kRows = 64u / LANES;   // of a wave
    static constexpr uint32_t kKeys = LANES * V, kRow = kKeys + std::max<uint32_t>(GF_ROUTE_MAX_GROUPS, LANES * kGap<V>);
    static constexpr uint32_t kIds = kRows * GF_ROUTE_MAX_K;
    static constexpr uint32_t kWave = kIds + std::max(kRows * kRow, 2u * kKeys);
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

// ---- sorted lists -------------------------------------------------------------
// An entry is a double whose upper word is its key's bits and whose lower one is
// its index, inverted under a positive key: doubles are ordered as floats are, by
// sign and magnitude, so the larger double is the larger key or, among equal
// keys, the lower index.  No key's bits reach a double's NaN (a float's infinity
// is a finite double), and no two entries are equal.
__device__ __forceinline__ double pack(float key, uint32_t index) {
    const uint32_t hi = __float_as_uint(key + 0.0f);   // -0 is 0
    const uint32_t lo = ~(index ^ uint32_t(int32_t(hi) >> 31));
    return __longlong_as_double((long long)(uint64_t(hi) << 32 | lo));
}
__device__ __forceinline__ float key_of(double e) {
    return __uint_as_float(uint32_t(uint64_t(__double_as_longlong(e)) >> 32));
}
__device__ __forceinline__ uint32_t index_of(double e) {
    const uint64_t u = uint64_t(__double_as_longlong(e));
    return ~(uint32_t(u) ^ uint32_t(int32_t(u >> 32) >> 31));
}
// Without the quieting of NaNs that fmax stands for.
__device__ __forceinline__ double larger(double a, double b) {
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double smaller(double a, double b) {
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ void in_order(double& a, double& b) {
    const double x = larger(a, b);
    b = smaller(a, b), a = x;
}
// Odd-even merge sort, largest first.
template <int N>
__device__ __forceinline__ void sort(double* a) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) in_order(a[i + j], a[i + j + k]);
}
// A list that falls and rises, largest first.
template <int N>
__device__ __forceinline__ void sort_bitonic(double* a) {
#pragma unroll
    for (int j = N / 2; j > 0; j /= 2)
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (!(i & j)) in_order(a[i], a[i | j]);
}
// The larger of two sorted lists' entries, at most LIST, sorted; `rest` the largest
// of those that go.
template <int LIST, int N>
__device__ __forceinline__ void join(const double* a, const double* b, double* to, bool want_rest, double& rest) {
    if constexpr (2 * N <= LIST) {
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = a[i], to[2 * N - 1 - i] = b[i];
        sort_bitonic<2 * N>(to);
    } else {
        if (want_rest) {
#pragma unroll
            for (int i = 0; i < N; ++i) rest = larger(rest, smaller(a[i], b[N - 1 - i]));
        }
        double top[N];
#pragma unroll
        for (int i = 0; i < N; ++i) top[i] = larger(a[i], b[N - 1 - i]);
        sort_bitonic<N>(top);
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = top[i];
    }
}
template <int LIST, int N>
constexpr int kJoined = 2 * N <= LIST ? 2 * N : LIST;
// Each lane's N entries, joined over the row's lanes: LIST of them in every lane.
template <int LIST, int CTRL, int N>
__device__ __forceinline__ void join_turned(double* a, bool want_rest, double& rest) {
    double b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) b[i] = dpp64<CTRL>(a[i]);
    if (want_rest) rest = larger(rest, dpp64<CTRL>(rest));
    double own[N];
#pragma unroll
    for (int i = 0; i < N; ++i) own[i] = a[i];
    join<LIST, N>(own, b, a, want_rest, rest);
}
template <bool HALVES>   // lanes ^ 32, or lanes ^ 16
__device__ __forceinline__ void both_sides(double v, double& a, double& b) {
    const uint64_t u = uint64_t(__double_as_longlong(v));
    const uint32_t lo = uint32_t(u), hi = uint32_t(u >> 32);
    uint32_t l[2], h[2];
    if constexpr (HALVES) {
        const auto x = __builtin_amdgcn_permlane32_swap(lo, lo, false, false), y = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
        l[0] = x[0], l[1] = x[1], h[0] = y[0], h[1] = y[1];
    } else {
        const auto x = __builtin_amdgcn_permlane16_swap(lo, lo, false, false), y = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
        l[0] = x[0], l[1] = x[1], h[0] = y[0], h[1] = y[1];
    }
    a = __longlong_as_double((long long)(uint64_t(h[0]) << 32 | l[0]));
    b = __longlong_as_double((long long)(uint64_t(h[1]) << 32 | l[1]));
}
template <int LIST, bool HALVES>
__device__ __forceinline__ void join_swapped(double* a, bool want_rest, double& rest) {
    double x[LIST], y[LIST];
#pragma unroll
    for (int i = 0; i < LIST; ++i) both_sides<HALVES>(a[i], x[i], y[i]);
    if (want_rest) {
        double p, q;
        both_sides<HALVES>(rest, p, q);
        rest = larger(p, q);
    }
    join<LIST, LIST>(x, y, a, want_rest, rest);
}
template <int LIST, int LANES, int N>
__device__ __forceinline__ void join_row(double* a, bool want_rest, double& rest) {
    constexpr int A = kJoined<LIST, N>, B = kJoined<LIST, A>, C = kJoined<LIST, B>;
    join_turned<LIST, 0x128, N>(a, want_rest, rest);
    join_turned<LIST, 0x124, A>(a, want_rest, rest);
    join_turned<LIST, 0x122, B>(a, want_rest, rest);
    join_turned<LIST, 0x121, C>(a, want_rest, rest);
    static_assert(kJoined<LIST, C> == LIST, "");
    if constexpr (LANES == 64) {
        join_swapped<LIST, false>(a, want_rest, rest);
        join_swapped<LIST, true>(a, want_rest, rest);
    }
}

// A lane holds V consecutive entries of its row.  For 4 to 16 choices it sorts
// its own into a list of LIST and the row's lanes join theirs, in four (six) steps
// whose cost does not depend on k: every lane ends with the row's list.  Else
// (LIST = 0) the row's best is taken k times: a lane keeps its three best at hand,
// the lowest lane that has the largest key has the lowest index too, and it looks
// through its V again only when all three are chosen and it had more.  Groups
// that are whole lanes are ranked from the lanes' two best, by moves between
// lanes; others through LDS.
//
// What bounds it is a row's chain of dependent steps in few waves, and how the
// blocks share the chip, not the bytes: 10,000 rows of 256 in 32 bits, k = 8 by
// logit, 4 of 16 groups kept, take 13 us and the launch that clears the load 1.4
// (21 by the loop), 16,384 rows by sigmoid and bias in 8 groups 22 (30); what they
// read takes 2 and 4.  The vector instructions (296 and 390 a row) would take 5
// and 10 spread over all compute units; waves wait for half of their cycles.  A
// unit holds one block of sixteen waves, which takes about as long whether others
// run or not: by logit 8192 rows (128 blocks) take 12.7 us, 16,384 (256) 15.2,
// 20,000 (313, two rounds) 24.  Blocks of sixteen waves hold every instance to 128
// registers: of some, 4 to 28 go to scratch (13 of lists of 16 at 256 entries).
// A whole wave for a row of more
// than 256 (8 or 16 entries a lane instead of 32 or 64, a quarter of the
// registers) took 28 us for 4 rows of 1008 where sixteen lanes took 71, 62 for
// 10,636 rows of 1018 where they took 73.
template <class T, int LANES, int V, int LIST>
__global__ __launch_bounds__(1024) void k_route(gf_route_opts o, const T* logits, uint32_t rows, uint32_t E,
                                                         uint64_t ld, const float* bias, int32_t* ids, float* weights,
                                                         int32_t* load) {
    extern __shared__ __align__(16) uint32_t lds[];
    using L = RouteLds<LANES, V>;
    constexpr uint32_t kRows = L::kRows;
    const uint32_t waves = blockDim.x >> 6;
    const uint32_t lane = threadIdx.x & 63u, c = lane % LANES, mine = lane / LANES, wave = threadIdx.x >> 6;
    const uint32_t first = c * V;
    uint32_t* count = lds;
    uint32_t* own = lds + L::kKeys + wave * L::kWave;
    int32_t* chosen = reinterpret_cast<int32_t*>(own) + mine * GF_ROUTE_MAX_K;
    float* keys = reinterpret_cast<float*>(own + L::kIds);
    float *mykeys = keys + mine * L::kRow, *myranks = mykeys + L::kKeys;
    if (load) {
        for (uint32_t e = threadIdx.x; e < E; e += blockDim.x) count[e] = 0;
        __syncthreads();
    }
    const bool by_score = bias || (o.groups > 1u && o.group_score == GF_GROUP_TOP2);
    const bool soft = o.score == GF_SCORE_SOFTMAX;
    // groups of whole lanes, `span` each
    const bool whole = o.groups > 1u && LANES == 16 && E == 16u * V && 16u % o.groups == 0;
    const uint32_t span = whole ? 16u / o.groups : 1u;
    const uint32_t gs = E / o.groups, magic = ((1u << 20) + gs - 1u) / gs;   // e / gs = e magic >> 20 below 1024

    for (uint64_t t0 = (uint64_t(blockIdx.x) * waves + wave) * kRows; t0 < rows;
         t0 += uint64_t(gridDim.x) * waves * kRows) {
        const bool row_ok = t0 + mine < rows;
        const uint64_t t = row_ok ? t0 + mine : rows - 1u;   // lanes without a row repeat the last, unstored
        const T* row = logits + t * ld;
        float key[V];
        load_row<LANES, V>(row, first, E, mykeys, key);
        float mx = kNone, top = 0.0f;   // top: the largest |bias|
        if (bias) {
            float b[V];
            load_row<LANES, V>(bias, first, E, mykeys, b);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                key[j] = b[j] > kNone ? key[j] : kNone;
                top = fmaxf(top, b[j] > kNone ? fabsf(b[j]) : 0.0f);
            }
            top = max_row<LANES>(top);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {   // fmaxf takes a NaN for -inf
            key[j] = fminf(fmaxf(key[j], kNone), kLargest);
            mx = fmaxf(mx, key[j]);
        }
        mx = max_row<LANES>(mx);
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
            z = sum_row<LANES>(sum);
        }
        // How far a 32-bit key k may be off.  Softmax: score s = e^v / z, v <= 0.  v and
        // its product with log2 e are rounded, so e^v is off by (2 |v| + 2) 2^-24 of
        // itself, z by the mean of that over the scores (the mean of |v| is at most
        // log E < 7) and (V + 6) 2^-24 for its sum, 1 / z, its product with e^v and
        // the sum with the bias by 2^-24 each: 2^-23 s (|v| + 14 + V / 2) in all.
        // |v| <= -log s as z >= 1, and s (c - log s) grows with s up to 1 for c >= 1: any
        // bound of s may stand for it, |k| + top or 1.  Sigmoid: the error of
        // e = e^-v weighs e / (1 + e)^2, below 1/4, which |v| times is below 0.23: 2^-24
        // in all; the sum, the reciprocal (2^-23) and the sum with the bias add 2^-22 of
        // the score and the key.  An infinite bias makes every bound of its row infinite, and
        // sigmoids around 2^-24 and below are all within theirs: such rows go through
        // the pass in 64 bits (16,384 x 256, 8 groups by two best: 30 us, with one
        // infinite bias 79, with all logits near -30 87).
        auto off = [&](float k) {
            const float u = fabsf(k) + top, s = fminf(u, 1.0f);
            return soft ? 0x1p-23f * (s * (14.0f + V / 2 - 0.6931472f * __builtin_amdgcn_logf(s + 0x1p-126f)) + u) + 0x1p-126f
                        : 0x1p-24f + 0x1p-22f * u;
        };
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
                load_row<LANES, V>(bias, first, E, mykeys, b);
#pragma unroll
                for (int j = 0; j < V; ++j) key[j] = key[j] > kNone ? key[j] + b[j] : kNone;
            }
        }
        bool close = false;   // a comparison that 32 bits do not decide
        constexpr int kOwn = V < LIST ? V : LIST > 0 ? LIST : 1;   // entries of the lane's own list
        double list[LIST > 0 ? LIST : 1], rest = pack(kNone, 0);
        Three best;
        // the lane's best entries of key[]
        auto gather = [&] {
            if constexpr (LIST > 0) {
                double all[V];
#pragma unroll
                for (int j = 0; j < V; ++j) all[j] = pack(key[j], first + j);
#pragma unroll
                for (int j = 0; j < V; j += kOwn) sort<kOwn>(all + j);
#pragma unroll
                for (int j = 0; j < kOwn; ++j) list[j] = all[j];
#pragma unroll
                for (int j = kOwn; j < V; j += kOwn) {
                    double own[kOwn];
#pragma unroll
                    for (int i = 0; i < kOwn; ++i) own[i] = list[i];
                    join<LIST, kOwn>(own, all + j, list, by_score, rest);
                }
            } else {
                best.clear();
#pragma unroll
                for (int j = 0; j < V; ++j) best.add(key[j], first + j);
            }
        };
        auto rank_of = [&](float first_best, float second_best) {
            return first_best + (o.group_score == GF_GROUP_TOP2 && second_best > kNone ? second_best : 0.0f);
        };
        // A rank is the sum of two keys at most, its rounding within their bounds; no
        // key is below -top, so neither is beyond |rank| + top.
        auto too_close = [&](float low, float high) {
            return by_score && high > kNone && low - high <= 2.0f * (off(fabsf(low) + top) + off(fabsf(high) + top));
        };
        if (o.groups == 1u || whole) {
            gather();
            if (whole) {
                float u, d;
                if constexpr (LIST > 0)
                    u = key_of(list[0]), d = V > 1 ? key_of(list[V > 1 ? 1 : 0]) : kNone;
                else
                    u = best.v[0], d = best.v[1];
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
                close = too_close(-max_row<LANES>(kept ? -rank : kNone), max_row<LANES>(kept ? kNone : rank));
                if constexpr (LIST > 0) {
#pragma unroll
                    for (int j = 0; j < kOwn; ++j) list[j] = kept ? list[j] : pack(kNone, 0);
                    rest = kept ? rest : pack(kNone, 0);
                } else if (!kept) {
                    best.clear();
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) mykeys[first + j] = key[j];
            wave_lds_sync();
            // `share` lanes a group, or up to four groups a lane; lanes start at
            // different places of their groups, in different banks
            const uint32_t wide = o.groups < uint32_t(LANES) ? 31u - uint32_t(__clz(int(LANES / o.groups))) : 0u;
            const uint32_t share = 1u << wide, p = c % share;
            for (uint32_t i = 0; i < o.groups; i += LANES >> wide) {
                const uint32_t g = i + (c >> wide);
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
            for (uint32_t i = 0; i < o.groups; i += LANES) {
                const uint32_t g = i + c;
                const float v = g < o.groups ? myranks[g] : kNone;
                uint32_t place = 0;
#pragma unroll 4
                for (uint32_t n = 0; n < o.groups; ++n) {
                    const float u = myranks[n];
                    place += u > v || (u == v && n < g);
                }
                const bool in = g < o.groups && place < o.keep_groups;
                kept |= ballot_row<LANES>(in) << i;
                if (in) low = fminf(low, v);
                else if (g < o.groups) high = fmaxf(high, v);
            }
            close = too_close(-max_row<LANES>(-low), max_row<LANES>(high));
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
            gather();
        }
        // the same logit and bias: an exact tie, the lower index first
        auto tied = [&](uint32_t a, uint32_t b) { return row[a] == row[b] && (!bias || bias[a] == bias[b]); };
        if constexpr (LIST > 0) {
            join_row<LIST, LANES, kOwn>(list, by_score, rest);
            // lane n has the list's entry n, and the one behind it
            double here = list[0], next = list[1];
#pragma unroll
            for (int n = 1; n < LIST; ++n) {
                here = c == uint32_t(n) ? list[n] : here;
                next = c == uint32_t(n) ? n + 1 < LIST ? list[n + 1 < LIST ? n + 1 : 0] : rest : next;
            }
            const float v = key_of(here), w = key_of(next);
            if (by_score && c < o.k && w > kNone && v - w <= off(v) + off(w))
                close |= !tied(index_of(here), index_of(next));
            if (c < o.k) chosen[c] = v > kNone ? int32_t(index_of(here)) : -1;
        } else {
            float before = 0.0f;
            bool more = best.v[2] > kNone;   // the lane may have a fourth
            for (uint32_t n = 0; n <= o.k; ++n) {
                const float m = max_row<LANES>(best.v[0]);
                const uint64_t who = ballot_row<LANES>(best.v[0] == m && m > kNone);
                if (by_score && n) {
                    bool near = who && before - m <= off(before) + off(m);
                    if (__any(near)) {
                        wave_lds_sync();
                        const uint32_t at = __shfl(best.i[0], int(mine * LANES + (who ? uint32_t(__ffsll((long long)who)) - 1u : 0u)));
                        if (near && tied(at, uint32_t(chosen[n - 1u]))) near = false;
                    }
                    close |= near;
                }
                before = m;
                if (n == o.k) break;
                if (!who && c == 0) chosen[n] = -1;
                if (who && c == uint32_t(__ffsll((long long)who)) - 1u) {
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
        }
        wave_lds_sync();
        if (by_score) {
            uint64_t again = __ballot(close);
            while (again) {
                const uint32_t r = uint32_t(__ffsll((long long)again) - 1) / LANES;
                again &= LANES == 64 ? 0u : ~(0xFFFFull << (r * 16u));   // the row's lanes
                choose_exact<(LANES * V + 63) / 64>(o, logits + min(t0 + r, uint64_t(rows) - 1u) * ld, E, bias, reinterpret_cast<double*>(keys),
                             reinterpret_cast<int32_t*>(own) + r * GF_ROUTE_MAX_K);
            }
        }
        constexpr uint32_t kChoices = GF_ROUTE_MAX_K / LANES;   // of the row, a lane, at most
        float s[kChoices], l[kChoices], sum = 0.0f, peak = kNone;
        int32_t id[kChoices];
#pragma unroll
        for (uint32_t i = 0; i < kChoices; ++i) {
            const uint32_t n = i * LANES + c;
            id[i] = n < o.k ? chosen[n] : -1;
            l[i] = id[i] >= 0 ? fminf(float(row[id[i]]), kLargest) : kNone;
            peak = fmaxf(peak, l[i]);
        }
        if (o.renormalise) mx = max_row<LANES>(peak);   // the softmax over the row cancels
        const float from = o.renormalise ? sigmoid_lift(mx) : 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kChoices; ++i) {
            s[i] = id[i] < 0 ? 0.0f : soft ? expf(l[i] - mx) / (o.renormalise ? 1.0f : z) : sigmoid(l[i], from);
            sum += s[i];
        }
        if (o.renormalise) sum = sum_row<LANES>(sum);
#pragma unroll
        for (uint32_t i = 0; i < kChoices; ++i) {
            const uint32_t n = i * LANES + c;
            if (!row_ok || n >= o.k) continue;
            ids[t * o.k + n] = id[i];
            weights[t * o.k + n] = o.scale * (o.renormalise ? sum > 0.0f ? s[i] / sum : 0.0f : s[i]);
            if (load && id[i] >= 0) atomicAdd(count + id[i], 1u);
        }
        wave_lds_sync();
    }
    if (load) {   // whole numbers: the order does not matter
        __syncthreads();
        for (uint32_t e = threadIdx.x; e < E; e += blockDim.x)
            if (gridDim.x == 1u)
                load[e] = int32_t(count[e]);
            else if (count[e])
                atomicAdd(load + e, int32_t(count[e]));
    }
}

__global__ void k_route_clear(int32_t* load, uint32_t E) {
    const uint32_t e = blockIdx.x * 256u + threadIdx.x;
    if (e < E) load[e] = 0;
}

// The gradient, sixteen lanes a row as above: the k chosen entries' terms are
// put into a row of LDS that is written out whole; the softmax over all
// entries adds its term to every live one.  16,384 rows of 256 in 32 bits, 8
// chosen: 7 us, 2.4 TB/s of gradient, bound by the chain from ids over logits to
// the sums; 15,287 rows of 992 with the softmax over all 57 us, 2.1 TB/s read and
// written, where the vector instructions would take 13: a block's 63.5 KB of LDS
// leave two waves a SIMD, which wait for 72% of their cycles.  Each exponential is
// taken once (twice took 2.4 times as long).
constexpr uint32_t kGradWaves = 4, kGradRows = 4;   // a block's waves, a wave's rows
template <class T>
__global__ __launch_bounds__(64 * kGradWaves) void k_route_grad(gf_route_opts o, const T* logits, uint32_t rows, uint32_t E,
                                                            uint64_t ld, const float* bias, const int32_t* ids,
                                                            const float* dweights, T* dlogits, uint64_t ldd) {
    extern __shared__ __align__(16) uint32_t lds[];
    const uint32_t lane = threadIdx.x & 63u, c = lane & 15u, wave = threadIdx.x >> 6;
    const uint32_t pitch = E + 7u & ~7u;
    float* d = reinterpret_cast<float*>(lds) + (wave * kGradRows + (lane >> 4)) * pitch;
    const bool soft = o.score == GF_SCORE_SOFTMAX;
    for (uint64_t t0 = (uint64_t(blockIdx.x) * kGradWaves + wave) * kGradRows; t0 < rows;
         t0 += uint64_t(gridDim.x) * kGradWaves * kGradRows) {
        const bool row_ok = t0 + (lane >> 4) < rows;
        const uint64_t t = row_ok ? t0 + (lane >> 4) : rows - 1u;
        const T* row = logits + t * ld;
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
#pragma unroll 4
            for (uint32_t e = c; e < E; e += 16u) {
                d[e] = entry(float(row[e]), bias, e);
                mx = fmaxf(mx, d[e]);
            }
            mx = max16(mx);
            const float lift = mx > kNone ? mx : 0.0f;
#pragma unroll 4
            for (uint32_t e = c; e < E; e += 16u) {   // a lane reads only what it wrote
                d[e] = expf(d[e] - lift);             // 0 for a masked entry
                z += d[e];
            }
            z = sum16(z);
        } else {
            mx = max16(peak), z = 1.0f;
        }
        const float from = o.renormalise ? sigmoid_lift(mx) : 0.0f;   // (sigmoids)
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            s[i] = id[i] < 0 ? 0.0f : soft ? expf(l[i] - mx) / z : sigmoid(l[i], from);
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
            for (uint32_t i = 0; i < 4u; ++i)   // below -17 a sigmoid's 1 - s is 1
                g[i] = o.scale * (g[i] - mean) * share[i] * (soft || l[i] < -17.0f ? 1.0f : 1.0f - s[i]);
        } else if (soft) {
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) mean += g[i] * s[i];
            mean = sum16(mean);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) g[i] *= o.scale * s[i] * (1.0f - s[i]);
        }
        if (all) {
            const float w = z > 0.0f ? -o.scale * mean / z : 0.0f;
#pragma unroll 4
            for (uint32_t e = c; e < E; e += 16u) d[e] = d[e] > 0.0f ? d[e] * w : 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) g[i] = o.scale * s[i] * (g[i] - mean);
        } else {
            for (uint32_t e = c * 4u; e < pitch; e += 64u) *reinterpret_cast<float4*>(d + e) = make_float4(0, 0, 0, 0);
        }
        wave_lds_sync();
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i)
            if (id[i] >= 0) d[id[i]] = g[i];
        wave_lds_sync();
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
// f(lanes a row, entries a lane)
template <class F>
hipError_t by_width(uint32_t E, F&& f) {
    constexpr std::integral_constant<int, 16> kPart;
    constexpr std::integral_constant<int, 64> kWave;
    if (E <= 16u) return f(kPart, std::integral_constant<int, 1>());
    if (E <= 32u) return f(kPart, std::integral_constant<int, 2>());
    if (E <= 64u) return f(kPart, std::integral_constant<int, 4>());
    if (E <= 128u) return f(kPart, std::integral_constant<int, 8>());
    if (E <= 256u) return f(kPart, std::integral_constant<int, 16>());
    if (E <= 512u) return f(kWave, std::integral_constant<int, 8>());
    return f(kWave, std::integral_constant<int, 16>());
}
// Beyond this many blocks a wave takes more than its first rows.
uint32_t route_blocks(uint64_t rows, uint32_t waves, uint32_t rows_of_wave) {
    return uint32_t(std::min<uint64_t>((rows + waves * rows_of_wave - 1u) / (waves * rows_of_wave), 8192u / waves));
}

}  // namespace

hipError_t launch_route(const gf_route_opts& opts, const MatIn& logits, uint32_t E, const float* bias, int32_t* ids,
                        float* weights, int32_t* load, hipStream_t st) {
    auto clear = [&] {
        if (load) hipLaunchKernelGGL(k_route_clear, dim3((E + 255u) / 256u), 256, 0, st, load, E);
        return hipGetLastError();
    };
    if (!logits.rows) return clear();
    gf_route_opts o = opts;
    // all groups: the same as none, but for GF_GROUP_TOP2's order by score
    if (o.keep_groups == o.groups && (bias || o.group_score == GF_GROUP_MAX)) o.groups = o.keep_groups = 1;
    return by_type(logits.dtype, [&](auto v) {
        return by_width(E, [&](auto lanes, auto width) {
            using T = decltype(v);
            constexpr int kLanes = decltype(lanes)::value, V = decltype(width)::value;
            using L = RouteLds<kLanes, V>;
            const uint64_t all = (logits.rows + L::kRows - 1u) / L::kRows;   // waves with rows
            // A block ends with an atomic addition for every entry that it counted: where
            // rows fill the chip anyway, few large blocks (4096 rows of 512 with the load
            // 16 us against 20, 10,000 of 512 25 against 37).  One block alone writes its
            // counts, and nothing need be cleared before it: 16 rows of 256, back to back 11.6
            // us against 14.2, a call alone 22.1 against 24.4 (64 rows, 16 waves: 26.1
            // against 24.6).
            const bool alone = load && all <= 8u;
            const uint32_t waves = alone ? uint32_t(all) : load && all >= 2048u ? 16u : 4u;
            if (!alone)
                if (const hipError_t e = clear()) return e;
            auto go = [&](auto lists) {
                hipLaunchKernelGGL((k_route<T, kLanes, V, decltype(lists)::value>),
                                   dim3(alone ? 1u : route_blocks(logits.rows, waves, L::kRows)), 64u * waves,
                                   4u * (L::kKeys + waves * L::kWave), st, o, static_cast<const T*>(logits.p),
                                   uint32_t(logits.rows), E, logits.ld, bias, ids, weights, load);
                return hipGetLastError();
            };
            // Lists cost the same for every k, a turn of the loop for every entry.  32,768
            // rows of 256 and of 896, by lists against the loop: k = 2 27.0 us against 27.8 and
            // 59 against 59, k = 8 27 against 37 and 64 against 88, k = 16 33 against 59 and
            // 86 against 119.
            if (o.k < 4u || o.k > 16u) return go(std::integral_constant<int, 0>());
            return o.k <= 8u ? go(std::integral_constant<int, 8>()) : go(std::integral_constant<int, 16>());
        });
    });
}

hipError_t launch_route_grad(const gf_route_opts& o, const MatIn& logits, uint32_t E, const float* bias,
                             const int32_t* ids, const float* dweights, const MatOut& dlogits, hipStream_t st) {
    return by_type(logits.dtype, [&](auto v) {
        using T = decltype(v);
        hipLaunchKernelGGL(k_route_grad<T>, dim3(route_blocks(logits.rows, kGradWaves, kGradRows)), 64 * kGradWaves,
                           kGradWaves * kGradRows * (E + 7u & ~7u) * 4u, st, o, static_cast<const T*>(logits.p),
                           uint32_t(logits.rows), E, logits.ld, bias, ids, dweights, static_cast<T*>(dlogits.p), dlogits.ld);
        return hipGetLastError();
    });
}

}  // namespace gf
