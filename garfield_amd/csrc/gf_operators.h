// Launchers of the operators on device memory (gf_mx.hip, gf_route.hip), which
// gf_operators.cpp checks arguments for.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/garfield.h"

namespace gf {

// A matrix of one of the three element types; ld in elements.
struct MatIn {
    const void* p;
    int32_t dtype;
    uint64_t rows, ld;
};
struct MatOut {
    void* p;
    int32_t dtype;
    uint64_t ld;
};

// Launchers return hipErrorInvalidConfiguration for sizes that need more
// threads than a launch has.
inline bool grid_fits(uint64_t blocks, uint32_t threads) { return blocks <= 0xFFFFFFFFu / threads; }

inline uint32_t mx_chunks(uint32_t K) { return (K >> 7) + ((K & 127u) != 0); }  // of 128 values a row

hipError_t launch_mx_quantise(const MatIn& x, uint32_t K, uint8_t* codes, uint8_t* scales, hipStream_t st);
hipError_t launch_mx_dequantise(const gf_mx_rows& w, const MatOut& out, hipStream_t st);
hipError_t launch_mx_product(const MatIn& x, const gf_mx_rows& w, const MatOut& out, void* ws, hipStream_t st);
hipError_t launch_mx_product_mx(const gf_mx_rows& x, const gf_mx_rows& w, const MatOut& out, void* ws,
                                hipStream_t st);
hipError_t launch_mx_product_grad(const MatIn& dy, const gf_mx_rows& w, const MatOut& dx, void* ws, hipStream_t st);
// Workspace bytes by kind (0 product, 1 both at four bits, 2 gradient): enough
// for M real rows wherever they lie, and those of one call (of x its address and
// row distance count, its values are not read).
size_t mx_workspace(int32_t kind, int32_t dtype, uint64_t M, uint64_t rows, uint32_t K);
size_t mx_workspace(int32_t kind, const MatIn& x, uint64_t rows, uint32_t K);

hipError_t launch_route(const gf_route_opts& o, const MatIn& logits, uint32_t E, const float* bias, int32_t* ids,
                        float* weights, int32_t* load, hipStream_t st);
hipError_t launch_route_grad(const gf_route_opts& o, const MatIn& logits, uint32_t E, const float* bias,
                             const int32_t* ids, const float* dweights, const MatOut& dlogits, hipStream_t st);

}  // namespace gf
