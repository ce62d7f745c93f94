// Both gradients of a product z = x W^T from the gradient d of z, in one launch: dx = d W and dW = d^T x, with the sums of d over its
// rows.  Each sum may be cut into parts, which leave sums of their own for another launch to add up.
#pragma once
#include "product_tile.h"

namespace vtdge {

// out = A B over a dimension that may be cut into several parts
struct GradArgs {
    Operand a, b;
    int64_t rows, cols, span_a, span_b, sum_a, sum_b;      // of the result; elements of a row of memory; rows of memory that may be read
    int tm, tn, stages, splits;
    float *part; int64_t part_stride; int accumulate;       // [splits], [rows][cols] fp32 each
    void *out;                                              // without `part`: the result, scaled; neither: only the sums
    float *sums_part; int64_t sums_stride; void *sums;     // nullable: the sums of A's rows, in the same way
};
struct GradPair {
    GradArgs dx, dw;
    int first_dw;                                           // workgroups before are dx's
    const float *scale, *scale2; int f32;                  // results in fp32
    bool f32_parts;                                         // operands in three bf16 parts
    // (not in parts) d has no rows of zeros behind its last, where dW's sum ends; the second operands lie with the summed dimension along
    // their rows, filled up with zeros to whole slabs
    bool ends;
};

// out = scale * (sum over the parts), for up to three results in one launch
struct SumJob {
    const float *part; void *out; int64_t n, stride; int parts;
};

// Shape and cuts of both gradients, the same for the same sizes.
struct GradPlan {
    int grads;                                      // shape
    int gm, gn, slab_g;                             // its tile and slab
    int dx_splits, dw_splits;
};
// (`ends`: of GradPair)
void plan_gradients(GradPlan &p, int64_t rows, int64_t classes, int width, bool split, bool ends);
// elements from one part of a sum to the next
inline int64_t part_of(int64_t n) { return (n + 63) / 64 * 64; }
// tm, tn and first_dw are filled in.  `what`: the entry point, for errors
int launch_gradients(const GradPlan &p, GradPair &g, const char *what, hipStream_t st);
// the parts of up to three sums added up
int sum_parts(const SumJob *jobs, int count, const float *scale, const float *scale2, bool f32, const char *what, hipStream_t st);

#define VT_STEP(call)                        \
    do {                                     \
        const int vt_rc = (call);            \
        if (vt_rc != VTDGE_OK) return vt_rc; \
    } while (0)

}  // namespace vtdge
