// Host side of gated_norm.hip.
#pragma once
#include <hip/hip_runtime_api.h>

namespace pdt {

struct GatedNorm {
    const __bf16 *x, *y;            // [M, D], M = B * T
    const float *gate, *w, *b;    // gate [D], or [B, D]
    const float *pw, *pb;         // norm after the branch, or null
    long M, T;
    int D;
    bool per_sample;
    float a, eps;
};
struct GatedNormPlan {
    int chunks, blocks;  // parts of a sample's rows; workgroups
    long units;          // samples * chunks
};

bool gated_norm_dim_ok(long D);
void launch_gated_norm_fwd(const GatedNorm& p, void* u, void* n, float* stats, hipStream_t s);
GatedNormPlan gated_norm_plan(long B, long T, long M, bool per_sample);
void launch_gated_norm_bwd(const GatedNorm& p, const GatedNormPlan& q, const void* du, const void* dn, const float* stats, void* dx,
                           void* dy, float* gate_part, long gate_stride, float* slab, int srow, hipStream_t s);
// sums [n] of the slab [rows][n] (or null), dgate [B][D] of the parts [B][chunks][D] (or null)
void launch_gated_norm_sums(const float* slab, float* sums, int rows, int n, const float* part, float* dgate, long B, int D, int chunks,
                            hipStream_t s);

}  // namespace pdt
