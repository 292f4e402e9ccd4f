// Products of real rows with 4-bit rows, and their gradient, on the bfloat16
// matrix instructions.
//
// A value of a 4-bit row is exact in bfloat16 at scale bytes up to 252 (at 253 and
// 254, which quantisation never writes, codes from 4 and 2 on become infinities),
// so only the real side could lose bits.  It does not: a binary16 value is the sum
// of two bfloat16 values, an fp32 value of three (truncated eight bits at a time;
// what lies below bfloat16's least, 2^-133, is cut off), and the product runs once
// over each of these planes.
#include <algorithm>

#include "gf_mx_device.h"

namespace gf {
namespace {

template <int DT>
constexpr int kPlanes = DT == GF_BF16 ? 1 : DT == GF_F16 ? 2 : 3;

// The planes of eight values: the leading 8 bits, the next 8, the last.  An
// infinity or NaN lies in the first alone (a NaN quieted, so that the upper half
// keeps a bit of its payload); no remainder exceeds the value, so none overflows.
template <int P>
__device__ __forceinline__ void split8(const float* v, uint4* plane) {
    uint32_t out[P][4];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        uint32_t top[P][2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float whole = __builtin_canonicalizef(v[i + k]);
            float rest = __builtin_isfinite(whole) ? whole : 0.0f;
            top[0][k] = __float_as_uint(whole);
#pragma unroll
            for (int p = 1; p < P; ++p) {
                rest -= __uint_as_float(__float_as_uint(rest) & 0xFFFF0000u);
                top[p][k] = __float_as_uint(rest);
            }
        }
#pragma unroll
        for (int p = 0; p < P; ++p) out[p][i / 2] = __builtin_amdgcn_perm(top[p][1], top[p][0], 0x07060302u);   // upper halves
    }
#pragma unroll
    for (int p = 0; p < P; ++p) plane[p] = make_uint4(out[p][0], out[p][1], out[p][2], out[p][3]);
}

// Eight elements of a row from k on, zeros from K on (WHOLE: all below K), as
// planes.
template <int DT, bool WHOLE = false>
__device__ __forceinline__ void load_planes(const ElemT<DT>* row, uint32_t k, uint32_t K, uint4* plane) {
    constexpr int P = kPlanes<DT>;
    ElemT<DT> e[8];
    if (WHOLE || k + 8u <= K) {
#pragma unroll
        for (uint32_t i = 0; i < sizeof(e) / 16u; ++i) {
            const uint4 q = load16(reinterpret_cast<const uint8_t*>(row + k) + i * 16u);
            __builtin_memcpy(reinterpret_cast<uint8_t*>(e) + i * 16u, &q, 16);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) e[i] = k + i < K ? row[k + i] : ElemT<DT>(0.0f);
    }
    if constexpr (DT == GF_BF16) {
        __builtin_memcpy(plane, e, 16);
    } else {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = float(e[i]);
        split8<P>(v, plane);
    }
}

// 8 codes to bfloat16.
__device__ __forceinline__ bf16x8 decode8(uint32_t codes, float scale) {
    bf16x8 o;
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1),
                 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
    o[0] = a[0], o[1] = a[1], o[2] = b[0], o[3] = b[1], o[4] = c[0], o[5] = c[1], o[6] = d[0], o[7] = d[1];
    return o;
}
__device__ __forceinline__ bf16x8 as_bf16x8(uint4 v) {
    bf16x8 o;
    __builtin_memcpy(&o, &v, 16);
    return o;
}

// ---- the real side as planes -----------------------------------------------
// planes[p][step][row][64]: a step's 64 values of all rows together, zeros from
// J on.  One pass, bound by memory: 4 (bfloat16) to 10 bytes a value.
template <int DT>
__global__ __launch_bounds__(256) void k_mx_planes(const ElemT<DT>* x, uint64_t rows, uint32_t J, uint64_t ld, uint32_t steps,
                                                   uint16_t* planes) {
    const uint32_t per = steps * 8u;
    const uint64_t n = rows * per;
    for (uint64_t i = uint64_t(blockIdx.x) * 256u + threadIdx.x; i < n; i += uint64_t(gridDim.x) * 256u) {
        const uint64_t r = n >> 32 ? i / per : uint32_t(i) / per;
        const uint32_t c = uint32_t(i - r * per);
        uint4 out[kPlanes<DT>];
        load_planes<DT>(x + r * ld, c * 8u, J, out);
#pragma unroll
        for (int p = 0; p < kPlanes<DT>; ++p)
            *reinterpret_cast<uint4*>(planes + ((uint64_t(p) * steps + c / 8u) * rows + r) * 64u + c % 8u * 8u) = out[p];
    }
}

// ---- few queries -----------------------------------------------------------
// Up to 16 queries: w is read once, straight to registers, and nothing else
// counts: one query in bfloat16 against 16384 rows of 4096 (37 MB) takes 9.4 us, 3.8
// TB/s, where loads of the same shape alone take 8.4.  A wave has 16 NT rows of w;
// the block's WK waves share them, each with its part of K, joined in order
// through LDS.  Lane group g of four holds block g of a chunk's four, 16 bytes;
// the values 8 q .. 8 q + 7 of the four blocks go through one instruction, on both
// sides alike.
template <int DT, int NT, int WK, int OT>
__global__ __launch_bounds__(64 * WK) void k_mx_few(const ElemT<DT>* x, uint32_t M, uint64_t ldx, gf_mx_rows w, uint32_t S,
                                                    ElemT<OT>* out, uint64_t ldo) {
    constexpr int P = kPlanes<DT>;
    __shared__ f32x4 part[WK > 1 ? WK * 64 * NT : 1];
    const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4, wk = threadIdx.x >> 6;
    const uint32_t N = uint32_t(w.rows), K = w.K, n0 = blockIdx.x * 16u * NT;
    f32x4 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = f32x4{0, 0, 0, 0};
    const uint8_t *wc[NT], *ws[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {   // rows beyond the end repeat the last one; their sums are not stored
        const uint64_t row = min(n0 + 16u * j + r, N - 1u);
        wc[j] = w.codes + row * S * 64u + g * 16u;
        ws[j] = w.scales + row * S * 4u;
    }
    const ElemT<DT>* xr = x + uint64_t(min(r, M - 1u)) * ldx;   // lanes without a query: the last again, not stored
    // Chunk s, byte[j] the scale byte of its block.
    auto chunk = [&](uint32_t s, const uint32_t* byte, auto whole) {
        uint4 c[NT], a[4][P];
#pragma unroll
        for (int j = 0; j < NT; ++j) c[j] = *reinterpret_cast<const uint4*>(wc[j] + uint64_t(s) * 64u);
#pragma unroll
        for (int q = 0; q < 4; ++q) load_planes<DT, decltype(whole)::value>(xr, s * 128u + g * 32u + q * 8u, K, a[q]);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const float scale = mx_scale(byte[j]);
            const uint32_t word[4] = {c[j].x, c[j].y, c[j].z, c[j].w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const bf16x8 b = decode8(word[q], scale);
#pragma unroll
                for (int p = 0; p < P; ++p)
                    acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, as_bf16x8(a[q][p]), acc[j], 0, 0, 0);
            }
        }
    };
    // Four whole chunks at a time: no branch stands between their loads, and a
    // row's scales come in one.  Then what is left, the last chunk perhaps cut.
    const uint32_t s1 = uint32_t(uint64_t(S) * (wk + 1u) / WK), cut = min(s1, K / 128u);
    uint32_t s = uint32_t(uint64_t(S) * wk / WK);
    for (; s + 4u <= cut; s += 4u) {
        uint4 sc[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) sc[j] = load16(ws[j] + uint64_t(s) * 4u);
#pragma unroll
        for (uint32_t u = 0; u < 4u; ++u) {
            uint32_t byte[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const uint32_t word[4] = {sc[j].x, sc[j].y, sc[j].z, sc[j].w};
                byte[j] = word[u] >> (8u * g) & 255u;
            }
            chunk(s + u, byte, std::true_type());
        }
    }
    for (; s < s1; ++s) {
        uint32_t byte[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) byte[j] = ws[j][uint64_t(s) * 4u + g];
        chunk(s, byte, std::false_type());
    }
    if (WK > 1) {
#pragma unroll
        for (int j = 0; j < NT; ++j) part[(wk * NT + j) * 64u + lane] = acc[j];
        __syncthreads();
        if (wk) return;
#pragma unroll
        for (int j = 0; j < NT; ++j)
            for (uint32_t k = 1; k < WK; ++k) acc[j] += part[(k * NT + j) * 64u + lane];
    }
    if (r < M) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
            for (uint32_t e = 0; e < 4u; ++e) {
                const uint32_t n = n0 + 16u * j + 4u * g + e;
                if (n < N) out[uint64_t(r) * ldo + n] = ElemT<OT>(acc[j][e]);
            }
    }
}

// ---- tiles through LDS -----------------------------------------------------
// A block has a tile of BM real rows x BN columns of the result, 64 values of
// the sum a step, its VM x VN waves equal parts of the tile.  The 4-bit side
// comes through registers, one block of 32 values a thread, decoded on its way
// to LDS, loaded one step ahead (two slots).  A real side in bfloat16 (or in
// planes, one after the other) comes by copies straight to LDS, two steps ahead
// (three slots; COPIED).  In tiles of 64 it comes through registers in its own
// type, split into its planes on its way, one step ahead (two slots): a small
// result is then one launch, whose rows need not be aligned or whole steps, and
// the planes share what is read and decoded of the other side.  A
// step has four parts; a part's operands are read from LDS while the part before
// it is multiplied, across steps too.
// Columns are rows of w (TR = false: the product) or positions in w's rows
// (TR = true: the gradient, whose sum runs over w's rows).  Slots of the real
// side, and of w without TR, have rows of 64 values, 128 bytes; their 16-byte
// piece c of row r lies at place c ^ (r / 2 & 7): rows take half the banks each
// by their parity, and of 16 rows the eight of one parity have a piece in eight
// different places.  With TR a slot has 64 rows of BN values as they lie in w
// and is read by the transposing LDS load, 4 rows x 16 columns a group of 16
// lanes; the 32-byte unit u of row n lies at place u ^ (n & 3), so that the
// four rows come from different banks.
// The sum may be cut into `parts`, each block then writing its own in fp32 to
// a workspace (out, rows of ldo, a part every M ldo), which k_mx_join adds up
// in order.
// 4096 x 8192 x 4096 in bfloat16 takes 222 us by tiles of 256 where calls follow one
// another (215 to 225 by the card), 1.24 PFLOP/s where the library's product of two
// bfloat16 matrices reaches 1.40 at 8192 x 8192 x 8192, the gradient 222 too; a call
// by itself 245, most under the profiler 235 to 258.  The matrix cores are busy for
// 45% of the cycles, at what the chip's power leaves of the clock.
template <int DT, bool COPIED, int BM, int BN, int OT, bool TR>
struct RealLds {
    static_assert(DT == GF_BF16 || !COPIED, "");
    static constexpr uint32_t kPlane = BM * 128u, kA = kPlane * kPlanes<DT>, kB = BN * 128u, kSlots = COPIED ? 3u : 2u;
    static constexpr uint32_t kBytes = kSlots * kA + 2u * kB;
    static constexpr uint32_t kCols = 32u;
    using P = Piece<OT, kCols>;
};

struct RealArgs {
    const void* a;       // the real side
    uint64_t lda, step;  // distance of its rows and, in bfloat16, steps, in elements
    uint32_t M, J;       // its rows, and their length
    uint32_t planes;     // in bfloat16: planes one after the other
    gf_mx_rows w;
    uint32_t S, N;       // N: columns of the result
    uint32_t tm, tn, parts;
};

template <int DT, bool COPIED, int BM, int BN, int VM, int VN, int OT, bool TR>
__global__ __launch_bounds__(64 * VM * VN) void k_mx_real(RealArgs p, ElemT<OT>* out, uint64_t ldo) {
    using L = RealLds<DT, COPIED, BM, BN, OT, TR>;
    using Pc = typename L::P;
    constexpr int P = kPlanes<DT>;
    constexpr uint32_t TH = 64u * VM * VN, kPer = BM * 8u / TH;   // 8-value pieces of the real side a thread and step
    constexpr int MI = BM / VM / 32, NI = BN / VN / 32;
    static_assert(BN * 2u == TH && VM * VN * Pc::kBytes <= L::kBytes, "");
    __shared__ __align__(16) uint8_t lds[L::kBytes];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, r = lane & 31u, h = lane >> 5;
    const uint32_t wave = uint32_t(__builtin_amdgcn_readfirstlane(int(tid >> 6)));
    const uint32_t base = lds_addr(lds);
    const uint32_t tiles = p.tm * p.tn, id = xcd_run(blockIdx.x, tiles * p.parts);
    const uint32_t cut = id / tiles;
    uint32_t m0, n0;
    tile_of(id % tiles, p.tm, p.tn, 4u, m0, n0);
    m0 *= BM, n0 *= BN;
    const uint32_t steps = (p.J + 63u) / 64u, total = steps * p.planes;
    const uint32_t s0 = uint32_t(uint64_t(total) * cut / p.parts), s1 = uint32_t(uint64_t(total) * (cut + 1u) / p.parts);

    // The thread's pieces: row i (TH / 8) + tid / 8, place tid & 7.  Rows beyond
    // the end repeat the last one; their sums are not stored.
    const uint32_t piece_of = (tid & 7u) ^ (tid >> 4 & 7u);
    uint32_t oa[kPer];                                   // byte offsets for the copies,
    const ElemT<DT>* ra[kPer];                           // or the rows
    constexpr uint32_t kRaw = sizeof(ElemT<DT>) / 2u;    // and eight values of each as loaded
    uint4 raw[kPer][kRaw];
    const uint8_t* pa = static_cast<const uint8_t*>(p.a) + uint64_t(m0) * p.lda * 2u;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        const uint32_t row = min(i * (TH / 8u) + tid / 8u, p.M - 1u - m0);
        if constexpr (!COPIED)
            ra[i] = static_cast<const ElemT<DT>*>(p.a) + uint64_t(m0 + row) * p.lda;
        else
            oa[i] = row * uint32_t(p.lda * 2u) + piece_of * 16u;
    }
    auto load_a = [&](uint32_t s, uint32_t slot) {
        if constexpr (COPIED) {
            const uint8_t* at = pa + uint64_t(s) * p.step * 2u;
#pragma unroll
            for (uint32_t i = 0; i < kPer; ++i) lds_copy16(at, oa[i], base + slot * L::kA + i * TH * 16u + wave * 1024u);
        } else {
            const uint32_t k = s * 64u + piece_of * 8u;
            if (k + 8u <= p.J) {
#pragma unroll
                for (uint32_t i = 0; i < kPer; ++i)
#pragma unroll
                    for (uint32_t q = 0; q < kRaw; ++q) raw[i][q] = load16(reinterpret_cast<const uint8_t*>(ra[i] + k) + q * 16u);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < kPer; ++i) {
                    ElemT<DT> e[8];
#pragma unroll
                    for (uint32_t c = 0; c < 8u; ++c) e[c] = k + c < p.J ? ra[i][k + c] : ElemT<DT>(0.0f);
                    __builtin_memcpy(raw[i], e, sizeof(e));
                }
            }
        }
    };
    auto write_a = [&](uint32_t slot) {
        if constexpr (!COPIED) {
#pragma unroll
            for (uint32_t i = 0; i < kPer; ++i) {
                uint4 plane[P];
                if constexpr (DT == GF_BF16) {
                    plane[0] = raw[i][0];
                } else {
                    ElemT<DT> e[8];
                    __builtin_memcpy(e, raw[i], sizeof(e));
                    float v[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c) v[c] = float(e[c]);
                    split8<P>(v, plane);
                }
#pragma unroll
                for (int q = 0; q < P; ++q)
                    *reinterpret_cast<uint4*>(lds + slot * L::kA + q * L::kPlane + (i * TH + tid) * 16u) = plane[q];
            }
        }
    };
    // A thread's block: row n0 + tid / 2, half tid & 1 of the step; with TR row
    // tid / (BN / 32) of the step, block tid % (BN / 32) of the tile's columns.
    constexpr uint32_t kAcross = BN / 32u;
    uint4 code;
    uint32_t byte;
    auto load_b = [&](uint32_t s) {
        const uint32_t j = s % steps;
        const uint64_t row = TR ? min(j * 64u + tid / kAcross, uint32_t(p.w.rows) - 1u) : min(n0 + tid / 2u, p.N - 1u);
        const uint64_t blk = row * (4u * p.S) + (TR ? min(n0 / 32u + tid % kAcross, 4u * p.S - 1u) : j * 2u + (tid & 1u));
        code = reinterpret_cast<const uint4*>(p.w.codes)[blk];
        byte = p.w.scales[blk];
    };
    auto write_b = [&](uint32_t slot) {
        uint8_t* to = lds + L::kSlots * L::kA + slot * L::kB;
        const float scale = mx_scale(byte);
        const uint32_t word[4] = {code.x, code.y, code.z, code.w};
#pragma unroll
        for (uint32_t q = 0; q < 4u; ++q) {
            const uint32_t row = TR ? tid / kAcross : tid / 2u;
            const uint32_t at = TR ? row * (BN * 2u) + ((tid % kAcross * 2u + q / 2u) ^ (row & 3u)) * 32u + q % 2u * 16u
                                   : row * 128u + (((tid & 1u) * 4u + q) ^ (row >> 1 & 7u)) * 16u;
            *reinterpret_cast<bf16x8*>(to + at) = decode8(word[q], scale);
        }
    };

    const uint32_t wm = wave / VN * (BM / VM), wn = wave % VN * (BN / VN);
    f32x16 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    // Values 16 q + 8 h .. of the step in slots sa and sb, into register set q & 1.
    bf16x8 a[2][P][MI], b[2][NI];
    auto read = [&](uint32_t sa, uint32_t sb, auto part) {
        constexpr uint32_t q = decltype(part)::value, set = q & 1u;
        const uint8_t *la = lds + sa * L::kA, *lb = lds + L::kSlots * L::kA + sb * L::kB;
        const uint32_t at = r * 128u + ((2u * q + h) ^ (r >> 1 & 7u)) * 16u;
#pragma unroll
        for (int c = 0; c < P; ++c)
#pragma unroll
            for (int i = 0; i < MI; ++i)
                a[set][c][i] = *reinterpret_cast<const bf16x8*>(la + c * L::kPlane + (wm + 32u * i) * 128u + at);
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            if constexpr (TR) {
                typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
                const uint32_t i = lane & 15u, row = 16u * q + 8u * h + (i >> 2);
                const uint32_t u = ((wn + 32u * j) / 16u + (lane >> 4 & 1u)) ^ (i >> 2);
                const uint8_t* from = lb + row * (BN * 2u) + u * 32u + (i & 3u) * 8u;
                const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)from);
                const bf16x4 hi =
                    __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(from + 4u * BN * 2u));
                b[set][j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            } else {
                b[set][j] = *reinterpret_cast<const bf16x8*>(lb + (wn + 32u * j) * 128u + at);
            }
        }
    };
    auto multiply = [&](auto part) {
        constexpr int set = decltype(part)::value & 1;
        sched_fence();
#pragma unroll
        for (int c = 0; c < P; ++c)
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b[set][j], a[set][c][i], acc[i][j], 0, 0, 0);
        sched_fence();
    };
    const std::integral_constant<int, 0> q0;
    const std::integral_constant<int, 1> q1;
    const std::integral_constant<int, 2> q2;
    const std::integral_constant<int, 3> q3;

    // The step in slots sa and sb, whose first part has been read; the next step
    // lies in the slots behind (after the last one: bytes that nothing uses).
    uint32_t sa = 0, sb = 0;
    auto step = [&]() {
        sched_fence();   // loads above start there, not where they are used
        read(sa, sb, q1);
        multiply(q0);
        read(sa, sb, q2);
        multiply(q1);
        read(sa, sb, q3);
        multiply(q2);
        lds_barrier();
        sa = sa + 1u == L::kSlots ? 0u : sa + 1u;
        sb ^= 1u;
        read(sa, sb, q0);
        multiply(q3);
    };
    auto load = [&](uint32_t s) {
        load_a(s, sa == 0 ? 2u : sa - 1u);   // (bfloat16) two slots on
        load_b(s);
    };
    auto landed = [&]() {   // the next step's; its slots are those of the step before,
        wait_vmcnt<0>();    // read out before the last barrier
        write_a(sa ^ 1u);
        write_b(sb ^ 1u);
    };

    // n >= 1 steps.  The first two are loaded together: a short sum waits for
    // memory once.
    const uint32_t n = s1 - s0;
    {
        const uint32_t next = min(s0 + 1u, s1 - 1u);
        load_a(s0, 0);
        load_b(s0);
        if constexpr (COPIED) load_a(next, 1);
        uint4 raw0[kPer][kRaw];
        __builtin_memcpy(raw0, raw, sizeof(raw));
        const uint4 code0 = code;
        const uint32_t byte0 = byte;
        if constexpr (!COPIED) load_a(next, 1);
        load_b(next);
        wait_vmcnt<0>();
        write_a(1);
        write_b(1);
        __builtin_memcpy(raw, raw0, sizeof(raw));
        code = code0, byte = byte0;
        write_a(0);
        write_b(0);
    }
    lds_barrier();
    if (n > 2u) load(s0 + 2u);
    read(0, 0, q0);
    step();
    for (uint32_t s = s0 + 1u; s + 2u < s1; ++s) {
        landed();
        load(s + 2u);
        step();
    }
    if (n > 2u) {
        landed();
        step();
    }
    if (n > 1u) step();
    wait_vmcnt<0>();
    lds_barrier();
    ElemT<OT>* o = out + uint64_t(cut) * p.M * ldo;
    uint8_t* piece = lds + wave * Pc::kBytes;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                Pc::put(piece, r, 8u * e + 4u * h,
                        f32x4{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]});
            wave_lds_sync();
            Pc::flush(piece, o, ldo, m0 + wm + 32u * i, n0 + wn + 32u * j, p.M, p.N);
            wave_lds_sync();
        }
}

// out = the sum of the parts, first to last, in fp32 (777 x 100 in 18 parts: 3.9 us,
// most of it the launch).
template <int OT>
__global__ __launch_bounds__(256) void k_mx_join(const float* part, uint32_t parts, uint64_t M, uint32_t N, ElemT<OT>* out,
                                                 uint64_t ldo) {
    const uint64_t n = M * N;
    for (uint64_t i = uint64_t(blockIdx.x) * 256u + threadIdx.x; i < n; i += uint64_t(gridDim.x) * 256u) {
        float v = part[i];
#pragma unroll 8
        for (uint32_t k = 1; k < parts; ++k) v += part[k * n + i];
        const uint64_t r = n >> 32 ? i / N : uint32_t(i) / N;
        out[r * ldo + (i - r * N)] = ElemT<OT>(v);
    }
}
// dx of no rows at all.
template <int OT>
__global__ __launch_bounds__(256) void k_mx_zero(uint64_t M, uint32_t N, ElemT<OT>* out, uint64_t ldo) {
    for (uint64_t i = uint64_t(blockIdx.x) * 256u + threadIdx.x; i < M * N; i += uint64_t(gridDim.x) * 256u)
        out[i / N * ldo + i % N] = ElemT<OT>(0.0f);
}

uint32_t blocks_for(uint64_t items) { return uint32_t(std::min<uint64_t>((items + 255u) / 256u, 1u << 20)); }

// How a product of M real rows of J values with N columns runs: the tile, the
// real side as planes or split in the kernel, and the sum in parts where the
// tiles leave compute units idle (up to six blocks a unit, at least four steps of
// 64 a part, and no more partial sums than 64 MiB).  The plan is part of the interface (the workspace's
// size), so it is made for the chip's compute units, not the current device's.
constexpr uint64_t kUnits = 256;
enum Tile { kLarge, kSmall, kSplit };
struct RealPlan {
    Tile tile;
    bool planes;   // the real side as planes in the workspace, not read in place or split
    uint32_t tm, tn, parts;
};
uint32_t planes_of(int32_t dtype) { return dtype == GF_BF16 ? 1u : dtype == GF_F16 ? 2u : 3u; }
// The plan is the one whose time, in us, is the least by this account: rounds of
// the chip's tiles, for each a step's time (one tile on a compute unit; two of
// the smaller ones) and once what a tile takes besides; a launch and 7 TB/s for
// planes and for joining parts, which are read back from the caches for the most
// part.  Fitted to 240 products and gradients of 17 to 10,000 real rows with each
// tile: four in five of its times are within 15% of the measured one, and the
// tile it takes was 1% slower than the best on average and 18% at most.  Parts up
// to one block a unit instead: the gradient of 4077 rows in fp32 over 5678 rows of
// 365 93 us against 75, 2759 over 31907 of 514 508 against 421.  Large,
// small, split: fp32, 4096 x 8192 x 4096 721, 867, 830 us, 2048 x 2048 x 4096 121, 153,
// 122; binary16, 1024 x 53124 x 1024 212, 222, 289, the gradient of 777 queries over
// 9376 rows of 100 38, 26, 19, in bfloat16 31, 23, 17; bfloat16, 4096 x 8192 x 4096
// 217, 275, 380, 64 x 53124 x 1024 31, 22, 17.
struct TileCost {
    float one, two, besides;
};
constexpr TileCost kTileCost[3][3] = {   // by tile, by type (GF_F32, GF_F16, GF_BF16)
    {{1.75f, 1.75f, 6.0f}, {1.51f, 1.51f, 6.0f}, {1.62f, 1.62f, 6.0f}},
    {{0.72f, 1.06f, 2.2f}, {0.65f, 1.00f, 2.2f}, {0.67f, 1.06f, 2.2f}},
    {{1.00f, 1.74f, 2.2f}, {0.85f, 1.30f, 2.0f}, {0.52f, 0.79f, 1.2f}}};
constexpr float kLaunch = 3.0f, kByte = 1.0f / 7e6f;
constexpr uint64_t kMostPlanes = 1ull << 32;   // bytes; beyond, the kernel splits and needs none
// in_place: the real side is read where it lies.
RealPlan real_plan(int32_t dtype, uint64_t M, uint64_t N, uint64_t J, bool in_place) {
    RealPlan best = {};
    float least = 0.0f;
    const uint64_t steps = (J + 63u) / 64u;
    for (const Tile tile : {kLarge, kSmall, kSplit}) {
        const uint64_t bm = tile == kLarge ? 256u : tile == kSmall ? 128u : 64u, bn = tile == kLarge ? 256u : 128u;
        const uint64_t tm = (M + bm - 1u) / bm, tn = (N + bn - 1u) / bn, planes = tile == kSplit ? 1u : planes_of(dtype);
        if (tile != kSplit && !in_place && M > kMostPlanes / (steps * planes * 128u)) continue;
        const TileCost& c = kTileCost[tile][dtype];
        const uint64_t round = tile == kLarge ? kUnits : 2u * kUnits;
        uint64_t last = 0;
        for (uint64_t units = kUnits; units <= 6u * kUnits; units += kUnits) {
            uint64_t parts = std::min<uint64_t>(units / (tm * tn), steps / 4u);
            parts = std::max<uint64_t>(std::min<uint64_t>(parts, (16u << 20) / (M * N)), 1u);
            if (parts == last) continue;
            last = parts;
            const uint64_t tiles = tm * tn * parts, full = tiles / round, rest = tiles % round;
            const float step = float(full) * c.two + (rest == 0 ? 0.0f : rest <= kUnits ? c.one : c.two);
            float us = step * float((steps * planes + parts - 1u) / parts) + c.besides * float(full + (rest != 0));
            if (tile != kSplit && !in_place)
                us += kLaunch + float(M) * float(J) * float(dtype == GF_F32 ? 10 : dtype == GF_F16 ? 6 : 4) * kByte;
            if (parts > 1u) us += kLaunch + float(M) * float(N) * float(parts) * 8.0f * kByte;
            if (best.tm && us >= least) continue;
            least = us;
            best = {tile, tile != kSplit && !in_place, uint32_t(tm), uint32_t(tn), uint32_t(parts)};
        }
    }
    return best;
}
// Whether a side of J values a row can be read in place: bfloat16, rows of whole
// steps, aligned for the copies.
bool in_place(int32_t dtype, const void* p, uint64_t ld, uint64_t J) {
    return dtype == GF_BF16 && J % 64u == 0 && ld % 8u == 0 && reinterpret_cast<uintptr_t>(p) % 16u == 0 && ld < 1u << 22;
}
size_t plan_bytes(const RealPlan& pl, int32_t dtype, uint64_t M, uint64_t N, uint64_t J) {
    return (pl.planes ? size_t((J + 63u) / 64u) * 128u * planes_of(dtype) * M : 0u) +
           (pl.parts > 1u ? size_t(pl.parts) * M * N * 4u : 0u);
}

template <bool TR>
hipError_t real_product(const MatIn& a, uint64_t J, const gf_mx_rows& w, uint64_t N, const MatOut& out, void* ws,
                        hipStream_t st) {
    const RealPlan pl = real_plan(a.dtype, a.rows, N, J, in_place(a.dtype, a.p, a.ld, J));
    if (!grid_fits(uint64_t(pl.tm) * pl.tn * pl.parts, 512u)) return hipErrorInvalidConfiguration;
    RealArgs p = {a.p, a.ld, 64, uint32_t(a.rows), uint32_t(J), 1u, w, mx_chunks(w.K), uint32_t(N), pl.tm, pl.tn, pl.parts};
    uint8_t* at = static_cast<uint8_t*>(ws);
    if (pl.planes) {
        const uint32_t steps = uint32_t((J + 63u) / 64u);
        p.a = at, p.lda = 64, p.step = a.rows * 64u, p.planes = planes_of(a.dtype);
        const hipError_t e = by_type(a.dtype, [&](auto dt) {
            constexpr int DT = decltype(dt)::value;
            hipLaunchKernelGGL(k_mx_planes<DT>, dim3(blocks_for(a.rows * steps * 8u)), 256, 0, st,
                               static_cast<const ElemT<DT>*>(a.p), a.rows, uint32_t(J), a.ld, steps,
                               reinterpret_cast<uint16_t*>(at));
            return hipGetLastError();
        });
        if (e != hipSuccess) return e;
        at += a.rows * steps * p.planes * 128u;
    }
    auto run = [&](auto ot, void* to, uint64_t ldo) {
        constexpr int OT = decltype(ot)::value;
        ElemT<OT>* o = static_cast<ElemT<OT>*>(to);
        const dim3 grid(pl.tm * pl.tn * pl.parts);
        if (pl.tile == kLarge)
            hipLaunchKernelGGL((k_mx_real<GF_BF16, true, 256, 256, 2, 4, OT, TR>), grid, 512, 0, st, p, o, ldo);
        else if (pl.tile == kSmall)
            hipLaunchKernelGGL((k_mx_real<GF_BF16, true, 128, 128, 2, 2, OT, TR>), grid, 256, 0, st, p, o, ldo);
        else if (a.dtype == GF_BF16)
            hipLaunchKernelGGL((k_mx_real<GF_BF16, false, 64, 128, 2, 2, OT, TR>), grid, 256, 0, st, p, o, ldo);
        else if (a.dtype == GF_F16)
            hipLaunchKernelGGL((k_mx_real<GF_F16, false, 64, 128, 2, 2, OT, TR>), grid, 256, 0, st, p, o, ldo);
        else
            hipLaunchKernelGGL((k_mx_real<GF_F32, false, 64, 128, 2, 2, OT, TR>), grid, 256, 0, st, p, o, ldo);
        return hipGetLastError();
    };
    if (pl.parts == 1u) return by_type(out.dtype, [&](auto ot) { return run(ot, out.p, out.ld); });
    if (const hipError_t e = run(std::integral_constant<int, GF_F32>(), at, N)) return e;
    return by_type(out.dtype, [&](auto ot) {
        constexpr int OT = decltype(ot)::value;
        hipLaunchKernelGGL(k_mx_join<OT>, dim3(blocks_for(a.rows * N)), 256, 0, st, reinterpret_cast<const float*>(at), pl.parts,
                           a.rows, uint32_t(N), static_cast<ElemT<OT>*>(out.p), out.ld);
        return hipGetLastError();
    });
}

constexpr uint64_t kFew = 16;   // queries that k_mx_few takes

}  // namespace

hipError_t launch_mx_product(const MatIn& x, const gf_mx_rows& w, const MatOut& out, void* ws, hipStream_t st) {
    if (x.rows > kFew) return real_product<false>(x, w.K, w, w.rows, out, ws, st);
    const uint32_t S = mx_chunks(w.K);
    return by_type(x.dtype, [&](auto dt) {
        return by_type(out.dtype, [&](auto ot) {
            constexpr int DT = decltype(dt)::value, OT = decltype(ot)::value;
            auto go = [&](auto nt, auto wk) {
                constexpr int NT = decltype(nt)::value, WK = decltype(wk)::value;
                if (!grid_fits((w.rows + 16u * NT - 1u) / (16u * NT), 64u * WK)) return hipErrorInvalidConfiguration;
                hipLaunchKernelGGL((k_mx_few<DT, NT, WK, OT>), dim3(uint32_t((w.rows + 16u * NT - 1u) / (16u * NT))), 64 * WK, 0,
                                   st, static_cast<const ElemT<DT>*>(x.p), uint32_t(x.rows), x.ld, w, S,
                                   static_cast<ElemT<OT>*>(out.p), out.ld);
                return hipGetLastError();
            };
            // Waves that fill the chip need not share K; where rows are few, they do.
            // A real side that is split takes more of a wave's time than the decoding,
            // so a split goes with more rows.  One query, <1, 1>, <2, 1>, <2, 4>, <1, 8>:
            // bfloat16, 53124 rows of 1024 8.3, 8.1, 13.6, 15.2 us, 16384 of 4096 14.2, 17.6,
            // 9.5, 10.6, 2000 of 8000 26, 33, 12, 8; binary16, <1, 1>, <4, 1>, <4, 4>, <4, 8>,
            // <2, 8>, <1, 8>: 300000 of 100 16, 11, 19, 37, 50, 78; 200000 of 2000 94, 80, 67,
            // 83, 98, 125; 16384 of 4096 24, 42, 16, 13, 14, 16; 8192 of 4096 21, 38, 15, 12,
            // 9, 10; 2000 of 8000 45, 74, 28, 20, 16, 13.
            const std::integral_constant<int, 1> one;
            const std::integral_constant<int, 2> two;
            const std::integral_constant<int, 4> four;
            const std::integral_constant<int, 8> eight;
            if constexpr (DT == GF_BF16) {
                if (w.rows >= 49152) return go(two, one);
                if (S >= 8 && w.rows >= 8192) return go(two, four);
            } else {
                if (w.rows >= 49152 && S <= 4) return go(four, one);
                if (w.rows >= 49152 || (w.rows >= 12288 && S >= 4 && S < 8)) return go(four, four);
                if (S >= 8 && w.rows >= 12288) return go(four, eight);
                if (S >= 8 && w.rows >= 4096) return go(two, eight);
            }
            if (S >= 8) return go(one, eight);
            return go(one, one);
        });
    });
}

hipError_t launch_mx_product_grad(const MatIn& dy, const gf_mx_rows& w, const MatOut& dx, void* ws, hipStream_t st) {
    if (w.rows) return real_product<true>(dy, w.rows, w, w.K, dx, ws, st);
    return by_type(dx.dtype, [&](auto ot) {
        constexpr int OT = decltype(ot)::value;
        hipLaunchKernelGGL(k_mx_zero<OT>, dim3(blocks_for(dy.rows * w.K)), 256, 0, st, dy.rows, w.K,
                           static_cast<ElemT<OT>*>(dx.p), dx.ld);
        return hipGetLastError();
    });
}

size_t mx_workspace(int32_t kind, int32_t dtype, uint64_t M, uint64_t rows, uint32_t K) {
    if (kind == 1 || !M || !rows || (kind == 0 && M <= kFew)) return 0;
    const uint64_t J = kind == 2 ? rows : K, N = kind == 2 ? K : rows;
    size_t most = plan_bytes(real_plan(dtype, M, N, J, false), dtype, M, N, J);
    if (in_place(dtype, nullptr, 0, J)) most = std::max(most, plan_bytes(real_plan(dtype, M, N, J, true), dtype, M, N, J));
    return most;
}
size_t mx_workspace(int32_t kind, const MatIn& x, uint64_t rows, uint32_t K) {
    if (kind == 1 || !x.rows || !rows || (kind == 0 && x.rows <= kFew)) return 0;
    const uint64_t J = kind == 2 ? rows : K, N = kind == 2 ? K : rows;
    return plan_bytes(real_plan(x.dtype, x.rows, N, J, in_place(x.dtype, x.p, x.ld, J)), x.dtype, x.rows, N, J);
}

}  // namespace gf
