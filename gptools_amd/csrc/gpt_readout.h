// Launchers of the read-out operators (internal): layer norm (gpt_norm.hip), the categorical log density of a linear
// read-out (gpt_class.hip). All memory is the caller's, workspaces included.
#pragma once
#include "../../include/gptools_hip.h"
#include <hip/hip_runtime.h>
#include <stdint.h>

struct NormArgs {
    const void *x, *weight, *bias, *ybar; // weight, bias may be null
    void *mean, *rstd;                    // written by the forward pass, read by the reverse one
    void *y, *xbar, *wbar, *bbar;         // wbar and bbar both null: not wanted
    void *partial, *partial2, *sums;      // workspace (partial), and parts of it
    int64_t rows, width, piece;
    unsigned column_blocks; // workgroups of columns before those of rows
    double eps;
};
size_t gpt_norm_workspace(int dtype, int64_t rows, int64_t width, bool vjp);
hipError_t gpt_launch_norm(int dtype, const NormArgs& a, hipStream_t st);
hipError_t gpt_launch_norm_vjp(int dtype, const NormArgs& a, hipStream_t st);

struct ClassArgs {
    const int64_t* y;                            // [rows] class of a row, < 0: not observed
    const void *x, *beta, *alpha;                // [rows][features], [classes][features], [classes] or null
    int64_t ldx, ldbeta, rows, features, classes; // row strides in elements
    const void* lpbar;                           // [rows] (Acc) or null: ones
    void *lp, *xbar, *alphabar, *betabar;        // alphabar may be null
    void* ws;
};
size_t gpt_class_workspace(int dtype, int64_t rows, int64_t features, int64_t classes, bool vjp);
hipError_t gpt_launch_class(int dtype, const ClassArgs& a, bool vjp, hipStream_t st);
// Few features (gpt_class_narrow.hip): what the two above turn to where it applies
bool gpt_class_narrow(int dtype, int64_t rows, int64_t features, int64_t classes, bool vjp);
size_t gpt_class_narrow_workspace(int dtype, int64_t rows, int64_t features, int64_t classes, bool vjp);
hipError_t gpt_launch_class_narrow(int dtype, const ClassArgs& a, bool vjp, hipStream_t st);
