// C entry points of the operators on device memory: argument checks, then one
// launcher each (gf_mx.hip, gf_route.hip).  Nothing here allocates or waits.
#include "gf_operators.h"

#include <limits>

#include "gf_state.h"

using gf::Error;

namespace {

template <class F>
gf_status guarded(F&& fn) {
    try {
        fn();
        return GF_OK;
    } catch (const Error& e) {
        gf::set_last_error(e.msg);
        return e.code;
    } catch (const std::bad_alloc&) {
        gf::set_last_error("host allocation failed");
        return GF_E_NOMEM;
    } catch (const std::exception& e) {
        gf::set_last_error(e.what());
        return GF_E_ARG;
    }
}

// Rows and columns stay below 2^31, so that kernels count them in 32 bits;
// offsets are 64-bit everywhere.
constexpr uint64_t kMaxRows = 0x7FFFFF00u;

void check_matrix(const void* p, int32_t dtype, uint64_t rows, uint64_t cols, uint64_t ld, const char* what) {
    GF_REQUIRE(dtype >= GF_F32 && dtype <= GF_BF16, GF_E_ARG, std::string(what) + ": unknown element type");
    GF_REQUIRE(rows <= kMaxRows && cols <= kMaxRows, GF_E_UNSUPPORTED, std::string(what) + ": more than 2^31 rows or columns");
    GF_REQUIRE(rows < 2 || ld >= cols, GF_E_ARG, std::string(what) + ": row distance below the row length");
    GF_REQUIRE(ld <= std::numeric_limits<uint64_t>::max() / 8 / (rows + 1), GF_E_ARG, std::string(what) + ": row distance too large");
    GF_REQUIRE(p || !rows || !cols, GF_E_ARG, std::string(what) + ": null pointer");
    GF_REQUIRE(reinterpret_cast<uintptr_t>(p) % (dtype == GF_F32 ? 4 : 2) == 0, GF_E_ARG, std::string(what) + ": pointer not aligned to its element");
}

void check_rows(const gf_mx_rows* w, const char* what) {
    GF_REQUIRE(w, GF_E_ARG, std::string(what) + ": null argument");
    GF_REQUIRE(w->K >= 1, GF_E_ARG, std::string(what) + ": K must be at least 1");
    GF_REQUIRE(w->rows <= kMaxRows && w->K <= kMaxRows, GF_E_UNSUPPORTED, std::string(what) + ": more than 2^31 rows or values a row");
    GF_REQUIRE((w->codes && w->scales) || !w->rows, GF_E_ARG, std::string(what) + ": null codes or scales");
    GF_REQUIRE(reinterpret_cast<uintptr_t>(w->codes) % 16 == 0 && reinterpret_cast<uintptr_t>(w->scales) % 4 == 0,
               GF_E_ARG, std::string(what) + ": codes must be aligned to 16 bytes, scales to 4");
}

void check_workspace(int32_t kind, const gf::MatIn& x, const gf_mx_rows& w, const void* ws, size_t bytes) {
    const size_t need = gf::mx_workspace(kind, x, w.rows, w.K);
    GF_REQUIRE(bytes >= need && (ws || !need), GF_E_ARG,
               "workspace of " + std::to_string(bytes) + " bytes, " + std::to_string(need) + " needed");
    GF_REQUIRE(!need || reinterpret_cast<uintptr_t>(ws) % 16 == 0, GF_E_ARG, "workspace must be aligned to 16 bytes");
}

void check_route(const gf_route_opts* o, uint64_t E, bool choose) {
    GF_REQUIRE(o, GF_E_ARG, "null options");
    GF_REQUIRE(E >= 1, GF_E_ARG, "E must be at least 1");
    GF_REQUIRE(E <= GF_ROUTE_MAX_E, GF_E_UNSUPPORTED, "E must be at most " + std::to_string(GF_ROUTE_MAX_E));
    GF_REQUIRE(o->k >= 1 && o->k <= E, GF_E_ARG, "k must be in 1..E");
    GF_REQUIRE(o->k <= GF_ROUTE_MAX_K, GF_E_UNSUPPORTED, "k must be at most " + std::to_string(GF_ROUTE_MAX_K));
    GF_REQUIRE(o->score == GF_SCORE_SOFTMAX || o->score == GF_SCORE_SIGMOID, GF_E_ARG, "unknown score");
    if (!choose) return;
    GF_REQUIRE(o->group_score == GF_GROUP_MAX || o->group_score == GF_GROUP_TOP2, GF_E_ARG, "unknown group score");
    GF_REQUIRE(o->groups >= 1 && E % o->groups == 0, GF_E_ARG, "groups must divide E");
    GF_REQUIRE(o->groups <= GF_ROUTE_MAX_GROUPS, GF_E_UNSUPPORTED, "groups must be at most " + std::to_string(GF_ROUTE_MAX_GROUPS));
    GF_REQUIRE(o->keep_groups >= 1 && o->keep_groups <= o->groups, GF_E_ARG, "keep_groups must be in 1..groups");
    GF_REQUIRE(o->k <= o->keep_groups * (E / o->groups), GF_E_ARG, "k exceeds the entries of keep_groups groups");
}

void launched(hipError_t e) {
    GF_REQUIRE(e != hipErrorInvalidConfiguration, GF_E_UNSUPPORTED, "sizes need more workgroups than a launch has");
    GF_HIP(e);
}

template <class T>
void check_pointer(const T* p, bool needed, const char* what) {
    GF_REQUIRE(p || !needed, GF_E_ARG, std::string(what) + ": null pointer");
    GF_REQUIRE(reinterpret_cast<uintptr_t>(p) % sizeof(T) == 0, GF_E_ARG, std::string(what) + ": pointer not aligned to its element");
}

}  // namespace

gf_status gf_mx_quantise(const void* x, int32_t dtype, uint64_t rows, uint32_t K, uint64_t ld, uint8_t* codes,
                         uint8_t* scales, void* stream) {
    return guarded([&] {
        check_matrix(x, dtype, rows, K, ld, "x");
        const gf_mx_rows out = {codes, scales, rows, K};
        check_rows(&out, "out");
        if (!rows) return;
        launched(gf::launch_mx_quantise({x, dtype, rows, ld}, K, codes, scales, hipStream_t(stream)));
    });
}

gf_status gf_mx_dequantise(const gf_mx_rows* w, int32_t dtype, void* out, uint64_t ldo, void* stream) {
    return guarded([&] {
        check_rows(w, "w");
        check_matrix(out, dtype, w->rows, w->K, ldo, "out");
        if (!w->rows) return;
        launched(gf::launch_mx_dequantise(*w, {out, dtype, ldo}, hipStream_t(stream)));
    });
}

gf_status gf_mx_product(const void* x, int32_t dtype, uint64_t M, uint64_t ldx, const gf_mx_rows* w, int32_t out_dtype,
                        void* out, uint64_t ldo, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_rows(w, "w");
        check_matrix(x, dtype, M, w->K, ldx, "x");
        check_matrix(out, out_dtype, M, w->rows, ldo, "out");
        check_workspace(0, {x, dtype, M, ldx}, *w, workspace, workspace_bytes);
        if (!M || !w->rows) return;
        launched(gf::launch_mx_product({x, dtype, M, ldx}, *w, {out, out_dtype, ldo}, workspace, hipStream_t(stream)));
    });
}

gf_status gf_mx_product_mx(const gf_mx_rows* x, const gf_mx_rows* w, int32_t out_dtype, void* out, uint64_t ldo,
                           void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_rows(x, "x");
        check_rows(w, "w");
        GF_REQUIRE(x->K == w->K, GF_E_ARG, "x and w hold different numbers of values a row");
        check_matrix(out, out_dtype, x->rows, w->rows, ldo, "out");
        check_workspace(1, {nullptr, GF_F32, x->rows, 0}, *w, workspace, workspace_bytes);
        if (!x->rows || !w->rows) return;
        launched(gf::launch_mx_product_mx(*x, *w, {out, out_dtype, ldo}, workspace, hipStream_t(stream)));
    });
}

gf_status gf_mx_product_grad(const void* dy, int32_t dtype, uint64_t M, uint64_t ldy, const gf_mx_rows* w,
                             int32_t out_dtype, void* dx, uint64_t ldo, void* workspace, size_t workspace_bytes,
                             void* stream) {
    return guarded([&] {
        check_rows(w, "w");
        check_matrix(dy, dtype, M, w->rows, ldy, "dy");
        check_matrix(dx, out_dtype, M, w->K, ldo, "dx");
        check_workspace(2, {dy, dtype, M, ldy}, *w, workspace, workspace_bytes);
        if (!M) return;
        launched(gf::launch_mx_product_grad({dy, dtype, M, ldy}, *w, {dx, out_dtype, ldo}, workspace,
                                          hipStream_t(stream)));
    });
}

gf_status gf_mx_product_workspace(int32_t kind, int32_t dtype, uint64_t M, uint64_t rows, uint32_t K, size_t* bytes) {
    return guarded([&] {
        GF_REQUIRE(bytes, GF_E_ARG, "null argument");
        GF_REQUIRE(kind >= 0 && kind <= 2, GF_E_ARG, "unknown kind");
        GF_REQUIRE(dtype >= GF_F32 && dtype <= GF_BF16, GF_E_ARG, "unknown element type");
        GF_REQUIRE(M <= kMaxRows && rows <= kMaxRows && K >= 1 && K <= kMaxRows, GF_E_ARG, "sizes out of range");
        *bytes = gf::mx_workspace(kind, dtype, M, rows, K);
    });
}

gf_status gf_mx_product_workspace_at(int32_t kind, const void* x, int32_t dtype, uint64_t M, uint64_t ldx, uint64_t rows,
                                     uint32_t K, size_t* bytes) {
    return guarded([&] {
        GF_REQUIRE(bytes, GF_E_ARG, "null argument");
        GF_REQUIRE(kind >= 0 && kind <= 2, GF_E_ARG, "unknown kind");
        GF_REQUIRE(dtype >= GF_F32 && dtype <= GF_BF16, GF_E_ARG, "unknown element type");
        GF_REQUIRE(M <= kMaxRows && rows <= kMaxRows && K >= 1 && K <= kMaxRows, GF_E_ARG, "sizes out of range");
        *bytes = gf::mx_workspace(kind, {x, dtype, M, ldx}, rows, K);
    });
}

gf_status gf_route(const gf_route_opts* opts, const void* logits, int32_t dtype, uint64_t T, uint32_t E, uint64_t ld,
                   const float* bias, int32_t* ids, float* weights, int32_t* load, void* stream) {
    return guarded([&] {
        check_route(opts, E, true);
        check_matrix(logits, dtype, T, E, ld, "logits");
        check_pointer(bias, false, "bias");
        check_pointer(ids, T != 0, "ids");
        check_pointer(weights, T != 0, "weights");
        check_pointer(load, false, "load");
        launched(gf::launch_route(*opts, {logits, dtype, T, ld}, E, bias, ids, weights, load, hipStream_t(stream)));
    });
}

gf_status gf_route_grad(const gf_route_opts* opts, const void* logits, int32_t dtype, uint64_t T, uint32_t E,
                        uint64_t ld, const float* bias, const int32_t* ids, const float* dweights, void* dlogits,
                        uint64_t ldd, void* stream) {
    return guarded([&] {
        check_route(opts, E, false);
        check_matrix(logits, dtype, T, E, ld, "logits");
        check_matrix(dlogits, dtype, T, E, ldd, "dlogits");
        check_pointer(bias, false, "bias");
        check_pointer(ids, T != 0, "ids");
        check_pointer(dweights, T != 0, "dweights");
        if (!T) return;
        launched(gf::launch_route_grad(*opts, {logits, dtype, T, ld}, E, bias, ids, dweights, {dlogits, dtype, ldd},
                                     hipStream_t(stream)));
    });
}
