// Products of 4-bit rows with 4-bit rows on the scaled matrix instructions.
//
// v_mfma_scale_f32_16x16x128 (32x32x64) takes from each lane one whole block
// of 32 values of one row, 16 bytes, and that block's scale byte: the format's
// blocks are the instruction's, so codes and scales go to it as they lie in
// memory.  w's rows are the first operand, so that a lane ends with four
// consecutive columns of the result.
#include <algorithm>

#include "gf_mx_device.h"

namespace gf {
namespace {

// One block of a row of each operand and the scale byte BYTE of its register.
template <int BYTE>
__device__ __forceinline__ f32x4 mfma16(uint4 a, uint32_t sa, uint4 b, uint32_t sb, f32x4 c) {
    const i32x8 x = {int(a.x), int(a.y), int(a.z), int(a.w)}, y = {int(b.x), int(b.y), int(b.z), int(b.w)};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, BYTE, int(sa), BYTE, int(sb));
}
template <int BYTE>
__device__ __forceinline__ f32x16 mfma32(uint4 a, uint32_t sa, uint4 b, uint32_t sb, f32x16 c) {
    const i32x8 x = {int(a.x), int(a.y), int(a.z), int(a.w)}, y = {int(b.x), int(b.y), int(b.z), int(b.w)};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 4, BYTE, int(sa), BYTE, int(sb));
}

// ---- operands straight from memory ----------------------------------------
// A wave has a tile of 16 MT queries x 16 NT rows.  The block's waves hold WN
// tiles side by side, and WK of them share a tile, each with its part of K,
// joined in order through LDS.  For few queries (all of w is read once, and
// what counts is the loads in flight), for short rows (the result is what
// takes the time) and for products too small for k_mx_tile's tiles.
// 10,000 x 62,500 x 128 to bfloat16 takes 271 us, 4.6 TB/s of result; the matrix cores
// are busy for 6% of it.  The result's rows are not whole lines: tiles side by
// side share one, and are dealt to one XCD in bands of eight (352, 319, 313,
// 305, 327, 360 us by bands of 1, 2, 4, 8, 16, 32 when that was chosen).
template <int MT, int NT, int WN, int WK, int OT>
__global__ __launch_bounds__(64 * WN * WK) void k_mx_direct(gf_mx_rows x, gf_mx_rows w, uint32_t S, uint32_t tm,
                                                            uint32_t tn, ElemT<OT>* out, uint64_t ldo) {
    constexpr uint32_t kJoin = WK > 1 ? WK * 64u * MT * NT * 16u : 0u;
    constexpr uint32_t kPieces = MT >= 2 && NT == 4 ? WN * Piece<OT, 64>::kBytes : 0u;
    __shared__ __align__(16) uint8_t lds[kJoin > kPieces ? kJoin : kPieces ? kPieces : 16u];
    const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
    const uint32_t wave = uint32_t(__builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)));
    const uint32_t wk = wave % WK, wn = wave / WK;
    const uint32_t M = uint32_t(x.rows), N = uint32_t(w.rows);
    uint32_t bm, bn;
    tile_of(xcd_run(blockIdx.x, tm * tn), tm, tn, 8u, bm, bn);
    const uint32_t m0 = bm * 16u * MT, n0 = (bn * WN + wn) * 16u * NT;
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    const uint8_t *xc[MT], *wc[NT], *xs[MT], *ws[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {   // rows beyond the end repeat the last one; their sums are not stored
        const uint64_t row = min(m0 + 16u * i + r, M - 1u);
        xc[i] = x.codes + row * S * 64u + g * 16u;
        xs[i] = x.scales + row * S * 4u + g;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const uint64_t row = min(n0 + 16u * j + r, N - 1u);
        wc[j] = w.codes + row * S * 64u + g * 16u;
        ws[j] = w.scales + row * S * 4u + g;
    }
    const uint32_t s1 = uint32_t(uint64_t(S) * (wk + 1u) / WK);
#pragma unroll 4
    for (uint32_t s = uint32_t(uint64_t(S) * wk / WK); s < s1; ++s) {
        uint4 a[MT], b[NT];
        uint32_t sa[MT], sb[NT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            a[i] = *reinterpret_cast<const uint4*>(xc[i] + uint64_t(s) * 64u);
            sa[i] = xs[i][uint64_t(s) * 4u];
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            b[j] = *reinterpret_cast<const uint4*>(wc[j] + uint64_t(s) * 64u);
            sb[j] = ws[j][uint64_t(s) * 4u];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = mfma16<0>(b[j], sb[j], a[i], sa[i], acc[i][j]);
    }
    if (WK > 1) {
        f32x4* part = reinterpret_cast<f32x4*>(lds) + uint32_t(wn * WK) * 64u * MT * NT;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) part[(wk * MT * NT + i * NT + j) * 64u + lane] = acc[i][j];
        __syncthreads();
        if (wk) return;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
                for (uint32_t k = 1; k < WK; ++k) acc[i][j] += part[(k * MT * NT + i * NT + j) * 64u + lane];
    }
    if constexpr (kPieces != 0) {
        uint8_t* piece = lds + wn * Piece<OT, 64>::kBytes;
        if (WK > 1) wave_lds_sync();   // WN is 1 then: the parts were read by this wave alone
#pragma unroll
        for (int i = 0; i < MT; i += 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < NT; ++j) Piece<OT, 64>::put(piece, 16u * h + r, 16u * j + 4u * g, acc[i + h][j]);
            wave_lds_sync();
            Piece<OT, 64>::flush(piece, out, ldo, m0 + 16u * i, n0, M, N);
            wave_lds_sync();
        }
    } else {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const uint32_t m = m0 + 16u * i + r, n = n0 + 16u * j + 4u * g;
                for (uint32_t e = 0; e < 4u; ++e)
                    if (m < M && n + e < N) out[uint64_t(m) * ldo + n + e] = ElemT<OT>(acc[i][j][e]);
            }
    }
}

// ---- operands through LDS --------------------------------------------------
// A block takes tiles of BM queries x BN rows one after another, its VM x VN
// waves equal parts of one, and a chunk of 128 values (4 blocks) of each row a
// step.  Steps, of all its tiles in one sequence, go through kSlots slots of
// LDS, filled by copies that pass no register: while a step is computed on,
// the next three are on the way.  A step has two parts; a part's operands are
// read from LDS while the part before it is multiplied, across steps too.
// Branches stand before a step's products only: the compiler moves matrix
// instructions down past a branch, and a barrier would then find the matrix
// cores idle.
// Of a row's 4 blocks lane group h (of two) takes blocks 2 h and 2 h + 1, on
// both sides alike: its scale bytes are then the low ones of a shifted word.
// The 16-byte block c of row r lies at place c ^ (r / 4 & 3) of the row: four
// rows of 64 bytes cover the banks, so of 16 rows the four that share banks
// have a block in four different places.
// Scales come 16 bytes a row, for four steps at once: a line is asked for once
// for four steps.  A tile's last group ends with the row (S >= 4), so that no
// read passes the end.  Groups are of four steps or, at the end of a tile,
// fewer, but never twice in a row: the four steps under way lie in three groups
// at most.
// 8192 x 8192 x 4096 to bfloat16 takes 147 us for quantised Gaussian rows, 3.7
// PFLOP/s, and 192 for codes drawn evenly: it is the chip's power that bounds it.
// The products alone take 85, as it holds them to 6.4 PFLOP/s, the copies alone
// 104; bands of 2, 4, 8, 16 tiles are alike.  Steps of 256 values in two slots took 190 us where these took 179, four
// waves of 128 x 128 211.
constexpr uint32_t kSlots = 4, kGroups = 3;

template <int BM, int BN, int OT>
struct TileLds {
    static constexpr uint32_t kRows = BM + BN, kSlot = kRows * 64u, kGroup = kRows * 16u;
    static constexpr uint32_t kBytes = kSlots * kSlot + kGroups * kGroup;
    static constexpr uint32_t kCols = OT == GF_F32 ? 16u : 32u;   // of a piece: 64-byte rows
    using P = Piece<OT, kCols>;
};

template <int BM, int BN, int VM, int VN, int OT>
__global__ __launch_bounds__(64 * VM * VN) void k_mx_tile(gf_mx_rows x, gf_mx_rows w, uint32_t S, uint32_t tm,
                                                          uint32_t tn, ElemT<OT>* out, uint64_t ldo) {
    using L = TileLds<BM, BN, OT>;
    using P = typename L::P;
    constexpr uint32_t TH = 64u * VM * VN, kRows = L::kRows, kSlot = L::kSlot;
    constexpr uint32_t kPer = kRows * 4u / TH, kPerS = kRows / TH;   // copies a thread and step, and group
    constexpr int MI = BM / VM / 32, NI = BN / VN / 32;
    static_assert(kRows % TH == 0 && TH % 64u == 0 && VM * VN * P::kBytes <= kSlot, "");
    __shared__ __align__(16) uint8_t lds[L::kBytes];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, r = lane & 31u, h = lane >> 5;
    const uint32_t wave = uint32_t(__builtin_amdgcn_readfirstlane(int(tid >> 6)));
    const uint32_t M = uint32_t(x.rows), N = uint32_t(w.rows), tiles = tm * tn;
    const uint32_t base = lds_addr(lds);
    auto corner = [&](uint32_t t, uint32_t& m0, uint32_t& n0) {
        tile_of(xcd_run(t, tiles), tm, tn, 4u, m0, n0);
        m0 *= BM, n0 *= BN;
    };

    // The copies' cursor: tile ft, step fs, scale group fg.  LDS row i of a
    // slot: query m0 + i, or row n0 + i - BM of w; beyond the ends the last row
    // again (its sums are not stored).
    uint32_t ft = blockIdx.x, fs = 0, fg = 0, oc[kPer], os[kPerS];
    const uint8_t *xc, *wc, *xs, *ws;   // of the tile's first row
    auto aim = [&]() {
        uint32_t m0, n0;
        corner(ft, m0, n0);
        xc = x.codes + uint64_t(m0) * S * 64u, wc = w.codes + uint64_t(n0) * S * 64u;
        xs = x.scales + uint64_t(m0) * S * 4u, ws = w.scales + uint64_t(n0) * S * 4u;
        auto row = [&](uint32_t i) { return i < BM ? min(i, M - 1u - m0) : min(i - BM, N - 1u - n0); };
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) oc[i] = row(i * (TH / 4u) + tid / 4u) * (S * 64u) + ((tid & 3u) ^ (tid >> 4 & 3u)) * 16u;
#pragma unroll
        for (uint32_t i = 0; i < kPerS; ++i) os[i] = row(i * TH + tid) * (S * 4u);
    };
    // Past the last tile the copies go on from the last one's rows, unused, so
    // that as many are always under way.
    auto fetch = [&](uint32_t slot) {
        if ((fs & 3u) == 0) {
            const uint32_t at = base + kSlots * kSlot + fg * L::kGroup;
            const uint32_t from = min(fs, S - 4u) * 4u;
#pragma unroll
            for (uint32_t i = 0; i < kPerS; ++i)
                lds_copy16((i * TH + wave * 64u < BM ? xs : ws) + from, os[i], at + i * TH * 16u + wave * 1024u);
            fg = fg + 1u == kGroups ? 0u : fg + 1u;
        }
        const uint32_t at = base + slot * kSlot;
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i)
            lds_copy16((i * (TH / 4u) < BM ? xc : wc) + uint64_t(fs) * 64u, oc[i], at + i * TH * 16u + wave * 1024u);
        if (++fs == S) {
            fs = 0;
            ft += gridDim.x;
            if (ft < tiles) aim();
        }
    };

    const uint32_t wm = wave / VN * (BM / VM), wn = wave % VN * (BN / VN);
    f32x16 acc[MI][NI];
    uint4 a[2][MI], b[2][NI];
    uint32_t sa[2][MI], sb[2][NI];
    uint32_t rs = 0, rg = kGroups - 1u;   // the step whose first part is read next, and its group's place
    // Part 0 or 1 of the step in `slot`.
    auto read = [&](uint32_t slot, auto part) {
        constexpr int B = decltype(part)::value;
        const uint8_t* p = lds + slot * kSlot;
        const uint32_t at = r * 64u + ((2u * h + B) ^ (r >> 2 & 3u)) * 16u;
#pragma unroll
        for (int i = 0; i < MI; ++i) a[B][i] = *reinterpret_cast<const uint4*>(p + (wm + 32u * i) * 64u + at);
#pragma unroll
        for (int j = 0; j < NI; ++j) b[B][j] = *reinterpret_cast<const uint4*>(p + (BM + wn + 32u * j) * 64u + at);
        if (B == 0) {
            if ((rs & 3u) == 0) rg = rg + 1u == kGroups ? 0u : rg + 1u;
            const uint32_t q = (rs | 3u) < S ? rs & 3u : rs - (S - 4u);   // the step's word in its group
            const uint8_t* g = lds + kSlots * kSlot + rg * L::kGroup + q * 4u;
#pragma unroll
            for (int i = 0; i < MI; ++i) sa[0][i] = *reinterpret_cast<const uint32_t*>(g + (wm + 32u * i + r) * 16u) >> (16u * h);
#pragma unroll
            for (int j = 0; j < NI; ++j) sb[0][j] = *reinterpret_cast<const uint32_t*>(g + (BM + wn + 32u * j + r) * 16u) >> (16u * h);
            rs = rs + 1u == S ? 0u : rs + 1u;
        } else {
#pragma unroll
            for (int i = 0; i < MI; ++i) sa[1][i] = sa[0][i];
#pragma unroll
            for (int j = 0; j < NI; ++j) sb[1][j] = sb[0][j];
        }
    };
    auto multiply = [&](auto part) {
        constexpr int B = decltype(part)::value;
        sched_fence();
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = mfma32<B>(b[B][j], sb[B][j], a[B][i], sa[B][i], acc[i][j]);
        sched_fence();
    };
    const std::integral_constant<int, 0> first;
    const std::integral_constant<int, 1> second;

    aim();
    fetch(0);
    fetch(1);
    fetch(2);
    wait_vmcnt<2u * kPer>();   // this wave's part of the first step has landed,
    lds_barrier();             // and the others'
    read(0, first);
    uint32_t slot = 0;
    for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
        for (uint32_t s = 0; s < S; ++s) {
            fetch((slot + 3u) % kSlots);   // the step before's slot, read out before the last barrier
            read(slot, second);
            multiply(first);
            wait_vmcnt<2u * kPer>();       // the next step's copies
            lds_barrier();
            slot = (slot + 1u) % kSlots;
            read(slot, first);             // after the last step of all: bytes that nothing uses
            multiply(second);
        }
        uint32_t m0, n0;
        corner(t, m0, n0);
        // the last step's slot is read out: the pieces' until the next copies
        uint8_t* piece = lds + (slot + 3u) % kSlots * kSlot + wave * P::kBytes;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int q = 0; q < int(32u / L::kCols); ++q) {
#pragma unroll
                    for (int e = 0; e < int(L::kCols / 8u); ++e) {
                        const int k = 4 * (e + q * int(L::kCols / 8u));
                        P::put(piece, r, 8u * e + 4u * h, f32x4{acc[i][j][k], acc[i][j][k + 1], acc[i][j][k + 2], acc[i][j][k + 3]});
                    }
                    wave_lds_sync();
                    P::flush(piece, out, ldo, m0 + wm + 32u * i, n0 + wn + 32u * j + L::kCols * q, M, N);
                    wave_lds_sync();
                }
        lds_barrier();   // every wave has read its last piece
    }
    wait_vmcnt<0>();   // no copy outlives the block
}

template <int MT, int NT, int WN, int WK>
hipError_t direct(const gf_mx_rows& x, const gf_mx_rows& w, const MatOut& out, hipStream_t st) {
    const uint32_t S = mx_chunks(w.K);
    const uint32_t tm = uint32_t((x.rows + 16u * MT - 1u) / (16u * MT)), tn = uint32_t((w.rows + 16u * NT * WN - 1u) / (16u * NT * WN));
    if (!grid_fits(uint64_t(tm) * tn, 64u * WN * WK)) return hipErrorInvalidConfiguration;
    return by_type(out.dtype, [&](auto ot) {
        constexpr int OT = decltype(ot)::value;
        hipLaunchKernelGGL((k_mx_direct<MT, NT, WN, WK, OT>), dim3(tm * tn), 64 * WN * WK, 0, st, x, w, S, tm, tn,
                           static_cast<ElemT<OT>*>(out.p), out.ld);
        return hipGetLastError();
    });
}
template <int BM, int BN, int VM, int VN>
hipError_t tile(const gf_mx_rows& x, const gf_mx_rows& w, const MatOut& out, hipStream_t st) {
    const uint32_t tm = uint32_t((x.rows + BM - 1u) / BM), tn = uint32_t((w.rows + BN - 1u) / BN);
    if (!grid_fits(uint64_t(tm) * tn, 64u * VM * VN)) return hipErrorInvalidConfiguration;
    return by_type(out.dtype, [&](auto ot) {
        constexpr int OT = decltype(ot)::value;
        // as many blocks as the chip's LDS holds at once
        const uint32_t blocks = std::min(tm * tn, compute_units() * (160u * 1024u / TileLds<BM, BN, OT>::kBytes));
        hipLaunchKernelGGL((k_mx_tile<BM, BN, VM, VN, OT>), dim3(blocks), 64 * VM * VN, 0, st, x, w, mx_chunks(w.K), tm,
                           tn, static_cast<ElemT<OT>*>(out.p), out.ld);
        return hipGetLastError();
    });
}

}  // namespace

hipError_t launch_mx_product_mx(const gf_mx_rows& x, const gf_mx_rows& w, const MatOut& out, void*, hipStream_t st) {
    const uint64_t M = x.rows, N = w.rows;
    const uint32_t S = mx_chunks(w.K);
    // Up to 16 queries: loads straight to registers, but many long rows come faster
    // by copies: direct against tiles, 16 x 53124 x 1024 14.5 us against 9.4, 5 x
    // 200000 x 2000 63 against 41; 16 x 16384 x 4096 11 against 15, 16 x 300000 x 640 29
    // against 32.
    if (M <= 16 && S >= 8 && N >= 32768 && S < 1u << 18) return tile<128, 128, 2, 2>(x, w, out, st);
    if (M <= 16) return S >= 8 ? direct<1, 1, 1, 8>(x, w, out, st) : direct<1, 1, 1, 1>(x, w, out, st);
    if (S >= 4 && S < 1u << 18) {
        if (large_tiles(M, N, compute_units())) return tile<256, 256, 2, 4>(x, w, out, st);
        // The tile of the least time by this account, in us: what a launch takes
        // besides, and for every chunk of K that of the blocks on a compute unit.
        // 32 x 32, 16 x 16, 32 x 64 and 128 x 128 measured: 17 x 2048 x 8192 14, 9, 23,
        // 26; 128 x 2048 x 8192 17, 30, 25, 25; 512 x 2048 x 8192 59, 114, 46, 25; 32 x
        // 53124 x 1024 19, 27, 14, 9; 26 x 1931 x 3352 6, 4, 9, 14; 500 x 500 x 1500 5, 7,
        // 7, 10.
        auto us = [&](uint64_t bm, uint64_t bn, float besides, float chunk) {
            const uint64_t blocks = ((M + bm - 1u) / bm) * ((N + bn - 1u) / bn);
            return besides + chunk * float(S) * std::max(1.0f, float(blocks) / 256.0f);
        };
        const float a = us(16, 16, 1.2f, 0.10f), b = us(32, 32, 2.0f, 0.20f), c = us(32, 64, 3.0f, 0.29f);
        if (us(128, 128, 6.0f, 0.31f) <= std::min(a, std::min(b, c))) return tile<128, 128, 2, 2>(x, w, out, st);
        if (a <= std::min(b, c)) return direct<1, 1, 1, 8>(x, w, out, st);
        if (b <= c) return direct<2, 2, 1, 8>(x, w, out, st);
    }
    if (S >= 4) return direct<2, 4, 1, 4>(x, w, out, st);
    return direct<4, 4, 4, 1>(x, w, out, st);
}

}  // namespace gf
