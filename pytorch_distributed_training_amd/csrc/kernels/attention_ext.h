// Host side of attention_ext.hip: operands, launch plans and launchers (the binding checks shapes and allocates).
#pragma once
#include <hip/hip_runtime_api.h>

#include "fastdiv.h"

namespace pdt {

// entries of a relative-position table that a head keeps in LDS: 16 KiB beside 66 of keys and codes at head_dim 128, where a CU's 160
// hold two workgroups up to 3584 entries and one above; four histograms of the gradient are 64 KiB
constexpr int kExtMaxEntries = 4096;

// rows of a [B, rows, heads, hd] tensor: element strides, and the division of a row by the heads that share a key head
struct ExtView {
    long bs, rs;
    FastDiv g;
};
struct ExtArgs {
    const __bf16 *q, *k, *v;
    ExtView qv, kv, o, dqv, dkv;  // k and v share strides; `o` holds for out and dout
    const int* lens;              // [B] valid keys, or null
    const float* tab;             // [H][Rp] bias per code difference, times sqrt(hd), or null
    const int *q_codes4, *k_codes4;  // byte offsets, padded to a multiple of 128
    const int2 *q_range, *k_range;   // smallest and largest of each 32
    int R, Rp;
    int self;                     // rows past lens[b] are dead too
    int B, Hkv, G, Sq, Sk, M, Mp; // M = Sq * G rows per key head, Mp = M rounded up to 64
    long stat_n;                  // B * Hkv * Mp: the statistics are [2][stat_n], -m and -log2 l
    float c, scale;               // log2(e) / sqrt(hd), 1 / sqrt(hd)
};
struct ExtPlan {
    bool few;  // one tile of rows per key head: the waves split the keys
    int tiles, splits;
};
struct ExtBwd {
    const void *out, *dout;
    const float* stat;
    float* dsum;  // [splits of the row owner][stat_n]: -D, in the end in the first
    float* ends;  // [ext_ends]: sums of dS over tiles of pairs past the table's reach, or null
    void *dq, *dk, *dv;
    float *part_q, *part_k, *part_v;
    ExtPlan q, kv;
};

ExtPlan ext_plan_fwd(long BH, int M, int Sk, bool bias);
void ext_plan_bwd(long BH, int M, int Sk, bool bias, ExtPlan& q, ExtPlan& kv);  // of the row owner and the key owner
// Floats of ExtBwd::ends, or 0 where the row owner need not sum pairs past the table's reach: with more positions than entries there
// are such pairs (positions in a row), with fewer (a grid) there are hardly any.  After ext_plan_bwd; with a gradient of the table.
long ext_ends(const ExtArgs& a, const ExtPlan& q);
void launch_ext_fwd(const ExtArgs& a, const ExtPlan& p, int hd, void* out, float* stat, float* part, float* part_ml,
                    hipStream_t s);
void launch_ext_bwd(const ExtArgs& a, const ExtBwd& w, int hd, hipStream_t s);
// codes [2 Sp + 4 Sp / 32]; position codes of 64 bits (wide) or 32
void launch_bias_tables(const float* table, const int* bucket_of, const void* q_codes, bool q_wide, const void* k_codes, bool k_wide,
                        float* tab, int* codes, int R, int Rp, int NB, int H, int S, int Sp, float inv_scale, hipStream_t s);
// the bias table's gradient: after launch_ext_bwd (which leaves D in dsum)
struct RelBlocks {
    int h0, heads, q0, qblocks, kblocks;  // of this launch: heads, blocks of 128 queries; blocks of 128 keys of all
    const float* ends;                    // of the row owner, or null
    int chunks, slab_rows;                // parts of the batch; rows of a head in the slab of entries
};
struct RelPlan {
    int heads, qblocks, chunks;  // of a launch
    int parts, rows;             // ranges of key tiles; slab rows per head
    long dense;                  // floats: sums of dS by pair
};
RelPlan rel_plan(int B, int H, int S, int hd);
// dense [plan.dense], slab [H][plan.rows][Rp], mid [H][Rp]
void launch_rel_bias_grad(const ExtArgs& a, const ExtBwd& w, int hd, const RelPlan& p, float* dense, float* slab, float* mid,
                          const int* bucket_of, float* dtable, int NB, hipStream_t s);

}  // namespace pdt
