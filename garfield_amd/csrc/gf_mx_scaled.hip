// Products of 4-bit rows with 4-bit rows on the scaled matrix instructions.
//
// v_mfma_scale_f32_16x16x128 (32x32x64) takes from each lane one whole block
// of 32 values of one row, 16 bytes, and that block's scale byte: the format's
// blocks are the instruction's, so codes and scales go to it as they lie in
// memory.  w's rows are the first operand, so that a lane ends with four
// consecutive columns of the result.
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
template <int MT, int NT, int WN, int WK, int OT>
__global__ __launch_bounds__(64 * WN * WK) void k_mx_direct(gf_mx_rows x, gf_mx_rows w, uint32_t S, uint32_t tm,
                                                            uint32_t tn, ElemT<OT>* out, uint64_t ldo) {
    constexpr uint32_t kJoin = WK > 1 ? WK * 64u * MT * NT * 16u : 0u;
    constexpr uint32_t kPieces = MT >= 2 && NT == 4 ? WN * Piece<OT>::kBytes : 0u;
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
        uint8_t* piece = lds + wn * Piece<OT>::kBytes;
        if (WK > 1) wave_lds_sync();   // WN is 1 then: the parts were read by this wave alone
#pragma unroll
        for (int i = 0; i < MT; i += 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < NT; ++j) Piece<OT>::put(piece, 16u * h + r, 16u * j + 4u * g, acc[i + h][j]);
            wave_lds_sync();
            Piece<OT>::flush(piece, out, ldo, m0 + 16u * i, n0, M, N);
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
// A block has a tile of BM queries x BN rows, its VM x VN waves equal parts of
// it, and takes 256 values (8 blocks, 128 bytes of codes) of each row a step.
// While one half of LDS is computed on, loads straight to LDS fill the other.
// Of a row's 8 blocks, lane group h (of two) takes blocks 4 h + s in step s,
// on both sides alike: its four scale bytes are then one word.  The 16-byte
// chunk c of row r lies at place c ^ (r & 7) of the row, so that eight
// consecutive rows read one chunk from eight different places.
template <int BM, int BN, int VM, int VN, int OT>
__global__ __launch_bounds__(64 * VM * VN) void k_mx_tile(gf_mx_rows x, gf_mx_rows w, uint32_t S, uint32_t tm,
                                                          uint32_t tn, ElemT<OT>* out, uint64_t ldo) {
    constexpr uint32_t TH = 64u * VM * VN, kRows = BM + BN, kCodes = kRows * 128u, kHalf = kCodes + kRows * 8u;
    constexpr uint32_t kPer = kRows * 8u / TH;    // 16-byte loads a thread and step
    constexpr uint32_t kPerS = kRows * 2u / TH;   // scale words a thread and step
    constexpr int MI = BM / VM / 32, NI = BN / VN / 32;
    constexpr uint32_t kPieces = VM * VN * Piece<OT>::kBytes;
    static_assert(NI == 2 && kRows * 2u % TH == 0, "");
    __shared__ __align__(16) uint8_t lds[2u * kHalf > kPieces ? 2u * kHalf : kPieces];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, r = lane & 31u, h = lane >> 5;
    const uint32_t wave = uint32_t(__builtin_amdgcn_readfirstlane(int(tid >> 6)));
    const uint32_t M = uint32_t(x.rows), N = uint32_t(w.rows);
    uint32_t bm, bn;
    tile_of(xcd_run(blockIdx.x, tm * tn), tm, tn, 4u, bm, bn);
    const uint32_t m0 = bm * BM, n0 = bn * BN;

    // LDS row i of a half: query m0 + i, or row n0 + i - BM of w; beyond the
    // ends the last row again (its sums are not stored).
    const uint8_t *pc[kPer], *ps[kPerS];
    auto row_at = [&](uint32_t i, uint32_t width, const uint8_t* cx, const uint8_t* cw) {
        return i < BM ? cx + uint64_t(min(m0 + i, M - 1u)) * S * width : cw + uint64_t(min(n0 + i - BM, N - 1u)) * S * width;
    };
    const uint32_t chunk = (tid & 7u) ^ (tid >> 3 & 7u);
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i)
        pc[i] = row_at(i * (TH / 8u) + tid / 8u, 64u, x.codes, w.codes) + chunk * 16u;
#pragma unroll
    for (uint32_t i = 0; i < kPerS; ++i)
        ps[i] = row_at(i * (TH / 2u) + tid / 2u, 4u, x.scales, w.scales) + (tid & 1u) * 4u;

    auto fetch = [&](uint32_t step, uint32_t half) {
        uint8_t* base = lds + half * kHalf;
        const bool whole = 2u * step + 2u <= S;
        if (whole || chunk < 4u) {
#pragma unroll
            for (uint32_t i = 0; i < kPer; ++i)
                __builtin_amdgcn_global_load_lds(
                    (const __attribute__((address_space(1))) void*)(pc[i] + uint64_t(step) * 128u),
                    (__attribute__((address_space(3))) void*)(base + i * TH * 16u + wave * 1024u), 16, 0, 0);
        } else {   // an odd last chunk of 128: the other half of the step is zeros
#pragma unroll
            for (uint32_t i = 0; i < kPer; ++i) *reinterpret_cast<uint4*>(base + (i * TH + tid) * 16u) = make_uint4(0, 0, 0, 0);
        }
        if (whole || !(tid & 1u)) {
#pragma unroll
            for (uint32_t i = 0; i < kPerS; ++i)
                __builtin_amdgcn_global_load_lds(
                    (const __attribute__((address_space(1))) void*)(ps[i] + uint64_t(step) * 8u),
                    (__attribute__((address_space(3))) void*)(base + kCodes + i * TH * 4u + wave * 256u), 4, 0, 0);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kPerS; ++i) *reinterpret_cast<uint32_t*>(base + kCodes + (i * TH + tid) * 4u) = 0u;
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

    auto part = [&](const uint8_t* base, const uint32_t* sa, const uint32_t* sb, auto byte) {
        constexpr int B = decltype(byte)::value;
        const uint32_t at = r * 128u + ((4u * h + B) ^ (r & 7u)) * 16u;
        uint4 a[MI], b[NI];
#pragma unroll
        for (int i = 0; i < MI; ++i) a[i] = *reinterpret_cast<const uint4*>(base + (wm + 32u * i) * 128u + at);
#pragma unroll
        for (int j = 0; j < NI; ++j) b[j] = *reinterpret_cast<const uint4*>(base + (BM + wn + 32u * j) * 128u + at);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = mfma32<B>(b[j], sb[j], a[i], sa[i], acc[i][j]);
    };

    const uint32_t steps = (S + 1u) / 2u;
    fetch(0, 0);
    for (uint32_t s = 0; s < steps; ++s) {
        __builtin_amdgcn_s_waitcnt(0x0F70);   // this wave's loads to LDS have landed
        __syncthreads();                      // and the others'; the other half has been read
        if (s + 1u < steps) fetch(s + 1u, (s + 1u) & 1u);
        const uint8_t* base = lds + (s & 1u) * kHalf;
        uint32_t sa[MI], sb[NI];
#pragma unroll
        for (int i = 0; i < MI; ++i)
            sa[i] = *reinterpret_cast<const uint32_t*>(base + kCodes + ((wm + 32u * i + r) * 2u + h) * 4u);
#pragma unroll
        for (int j = 0; j < NI; ++j)
            sb[j] = *reinterpret_cast<const uint32_t*>(base + kCodes + ((BM + wn + 32u * j + r) * 2u + h) * 4u);
        part(base, sa, sb, std::integral_constant<int, 0>());
        part(base, sa, sb, std::integral_constant<int, 1>());
        part(base, sa, sb, std::integral_constant<int, 2>());
        part(base, sa, sb, std::integral_constant<int, 3>());
    }
    __syncthreads();
    uint8_t* piece = lds + wave * Piece<OT>::kBytes;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                Piece<OT>::put(piece, r, 32u * j + 8u * e + 4u * h,
                               f32x4{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]});
        wave_lds_sync();
        Piece<OT>::flush(piece, out, ldo, m0 + wm + 32u * i, n0 + wn, M, N);
        wave_lds_sync();
    }
}

template <int MT, int NT, int WN, int WK>
hipError_t direct(const gf_mx_rows& x, const gf_mx_rows& w, const MatOut& out, hipStream_t st) {
    const uint32_t S = mx_chunks(w.K);
    const uint32_t tm = uint32_t((x.rows + 16u * MT - 1u) / (16u * MT)), tn = uint32_t((w.rows + 16u * NT * WN - 1u) / (16u * NT * WN));
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
    return by_type(out.dtype, [&](auto ot) {
        constexpr int OT = decltype(ot)::value;
        hipLaunchKernelGGL((k_mx_tile<BM, BN, VM, VN, OT>), dim3(tm * tn), 64 * VM * VN, 0, st, x, w, mx_chunks(w.K), tm,
                           tn, static_cast<ElemT<OT>*>(out.p), out.ld);
        return hipGetLastError();
    });
}

}  // namespace

hipError_t launch_mx_product_mx(const gf_mx_rows& x, const gf_mx_rows& w, const MatOut& out, void*, hipStream_t st) {
    const uint64_t M = x.rows, N = w.rows;
    const uint32_t S = mx_chunks(w.K);
    if (M <= 16) return S >= 8 ? direct<1, 1, 1, 8>(x, w, out, st) : direct<1, 1, 1, 1>(x, w, out, st);
    if (S >= 4) {
        const uint64_t big = ((M + 255) / 256) * ((N + 255) / 256), mid = ((M + 127) / 128) * ((N + 127) / 128);
        if (big >= 192) return tile<256, 256, 2, 4>(x, w, out, st);
        if (mid >= 128) return tile<128, 128, 2, 2>(x, w, out, st);
        return direct<4, 4, 1, 4>(x, w, out, st);
    }
    return direct<4, 4, 4, 1>(x, w, out, st);
}

}  // namespace gf
