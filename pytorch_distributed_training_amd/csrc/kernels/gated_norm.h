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
    // u and dx, which the model reads again a branch later, are stored past the caches: from 64 MB a tensor on (64 x 577 x 1024, 76 MB:
    // 155 -> 147 us forward and backward, ViT-B/16 with layer scale at batch 256 6470 -> 6492 images/s; at batch 64, 19 MB, it was
    // 4733 -> 4718).  n and dy are read at once: past the caches too they cost that model 0.4 to 0.9 %.
    bool stream;
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
