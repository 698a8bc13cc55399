// Attention of queries over keys that are laid out apart from them (forward + backward) on the gfx950 matrix cores:
// any two lengths, query heads that share a key head, valid key counts per sequence, and an additive bias that is learned
// per bucket of relative positions.  One family serves self attention with such a bias (packed projection, strided views)
// and cross attention to an encoder's states.
//
//   row r of a key head = (query position q = r / G, head g = r % G of its G query heads), M = Sq * G rows
//   S[r, j]  = c (q_r . k_j) + bias(q, j) log2(e),  c = log2(e) / sqrt(hd)      (scores in base 2)
//   P        = 2^(S - m) / l,  O = P V,  m = max_j S,  l = sum_j 2^(S - m)        j < len[b]; a row without keys is zero
//   dS       = P (dO V^T - D),  D = sum_j P_rj (dO V^T)_rj = dO_r . O_r
//   dQ       = dS K / sqrt(hd),  dK = dS^T Q / sqrt(hd),  dV = P^T dO  (the sum over r runs over the G heads too)
//
// The bias of (q, j) is tab[clamp(q_code[q] - k_code[j], 0, R-1)], a table of R floats per head in LDS: a position is one
// integer, so neither an [S, S] index nor an [H, S, S] bias is ever read.
//
//  * Scores are produced TRANSPOSED in the passes that own rows (lane = row, registers = keys) and straight in the pass that
//    owns keys (lane = key, registers = rows); the second product is transposed as well (V^T P^T, K^T dS^T, ...), so that
//    running maximum, sums, rescaling and the stores (four neighbouring channels a lane) are all per lane.
//  * The statistics that the backward gets are -m (in units of q . k) and -log2 l apart.  Where a bias of -1e9 holds for a whole
//    row, their sum would not leave a bit of l, and 2^(c s - sum), a difference of two numbers rounded at 1e9, is anything.
//  * With a bias the scores of both directions start at the bias and m is taken off the result, so that the backward's P are the
//    forward's to 32 bits: at -1e9 the bias takes up all of q . k, the keys of such a row weigh the same, and they have to weigh
//    the same in the gradients (with scores that start at bias - m a row's P added up to 1.2 to 2.8).
//  * The axis that streams comes by LDS-DMA in blocks of 64 rows, two buffers, one barrier a block; rows past the valid
//    length are sent out of range and arrive as zeros, so whatever they hold (NaN, infinities) is never multiplied.
//  * Few rows: the streamed axis is cut into `splits`, each with its own workgroup and an fp32 partial that a small kernel
//    joins in a fixed order.
//  * No atomics in memory: the bias gradient sums dS over the batch in registers first (a kernel of its own, which walks over
//    the batch with a block of pairs fixed), then the pairs by entry in a histogram per WAVE in LDS (program order), then waves
//    and workgroups in a fixed order.
#include <stdexcept>
#include <string>

#include "attn_tile.h"
#include "attention_ext.h"

namespace pdt {
namespace {

constexpr float kInf = __builtin_inff();
// Finite biases stay finite times sqrt(hd), and apart: from 2^120 on in magnitude what is over counts a sixteenth (lower stays lower
// by at least 2^92, equal stays equal; the type's lowest value, 2^128, becomes 2^124).  -inf stays -inf: never attended.
constexpr float kBiasFull = 0x1p120f;
__device__ __forceinline__ float finite_bias(float v) {
    const float over = fabsf(v) - kBiasFull;
    return over > 0.f && over < kInf ? copysignf(fmaf(over, 0.0625f, kBiasFull), v) : v;
}

// one 4-byte-aligned 16-B piece per lane into LDS (lane-linear), descriptor from wave-uniform words
__device__ __forceinline__ i32x4 uniform_rsrc(const void* base, uint32_t bytes) {
    i32x4 r = make_rsrc_words(base, bytes);
#pragma unroll
    for (int k = 0; k < 3; ++k) r[k] = __builtin_amdgcn_readfirstlane(r[k]);
    return r;
}
// every outstanding DMA and LDS access of this wave is done, and every wave is here; no memory access moves across
__device__ __forceinline__ void dma_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ int xcd_order(int id, int n) {
    // workgroup id runs on XCD id % 8: neighbours in the result (which read the same keys) get the same XCD and its L2
    const int q = n >> 3, r = n & 7, x = id & 7;
    return x * q + (x < r ? x : r) + (id >> 3);
}

// rows [r0, r0 + 64) of a matrix -> LDS image; rows >= valid arrive as zeros.  `off(row)` = element offset of row r0 + row
template <int HD, int NW, typename F>
__device__ __forceinline__ void dma_block(uint32_t img, const bf16* base, uint32_t bytes, int valid, int wave, int lane, F off) {
    using G = AttnGeo<HD>;
    constexpr int RPP = 1024 / G::ROWBYTES, NP = 64 / RPP;
    const i32x4 rsrc = uniform_rsrc(base, bytes);
#pragma unroll
    for (int i = 0; i < (NP + NW - 1) / NW; ++i) {
        const int p = wave + i * NW;
        if (NP % NW == 0 || p < NP) {
            const int row = p * RPP + lane / G::NCH;
            const int x = ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)) & (G::NCH - 1);
            const uint32_t o = row < valid ? (uint32_t)off(row) * 2u + (uint32_t)(((lane % G::NCH) ^ x) << 4) : kOOB;
            lds_dma16(rsrc, o, (uint32_t)__builtin_amdgcn_readfirstlane((int)(img + (uint32_t)p * 1024u)));
        }
    }
}
// rows [r0, r0 + 32) -> LDS image, by one wave; rows >= valid arrive as zeros.  STREAM: past the caches (streams_past_caches)
template <int HD, bool STREAM>
__device__ __forceinline__ void dma_tile(uint32_t img, const bf16* base, int rs, int valid, int lane) {
    using G = AttnGeo<HD>;
    constexpr int RPP = 1024 / G::ROWBYTES, NP = 32 / RPP;
    const i32x4 rsrc = uniform_rsrc(base, (uint32_t)(valid - 1) * (uint32_t)rs * 2u + G::ROWBYTES);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int row = p * RPP + lane / G::NCH;
        const int x = ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)) & (G::NCH - 1);
        const uint32_t o = row < valid ? (uint32_t)(row * rs) * 2u + (uint32_t)(((lane % G::NCH) ^ x) << 4) : kOOB;
        const uint32_t at = (uint32_t)__builtin_amdgcn_readfirstlane((int)(img + p * 1024));
        if (STREAM) lds_dma16_stream(rsrc, o, at);
        else lds_dma16(rsrc, o, at);
    }
}
// 64 consecutive 4-byte values -> LDS (the image takes 1 KiB: lanes 16.. write zeros)
__device__ __forceinline__ void dma_words(uint32_t img, const void* base, int lane) {
    lds_dma16(uniform_rsrc(base, 256u), lane < 16 ? (uint32_t)lane * 16u : kOOB, (uint32_t)__builtin_amdgcn_readfirstlane((int)img));
}

// LDS address of a pair's bias: clamp(q code - k code) in bytes, `lo` and `hi` the addresses of the table's first and last
// entry and `lo` already in the query's code (two instructions an element; a clamp of unknown bounds compiles to four)
__device__ __forceinline__ int bias_at(int qc4, int kc4, int lo, int hi) {
    int d = qc4 - kc4;
    asm("v_med3_i32 %0, %0, %1, %2" : "+v"(d) : "v"(lo), "s"(hi));
    return d;
}
typedef const float __attribute__((address_space(3))) * lds_cfloat_ptr;
__device__ __forceinline__ float lds_float(int addr) { return *(lds_cfloat_ptr)(uintptr_t)(uint32_t)addr; }

// The one table address that all pairs of 32 queries and 32 keys fall on, or -1: from the smallest and largest code of each side.
// Positions further apart than the table reaches share an entry, so on long sequences most tiles need no histogram.  (In the
// attention kernels the test cost more than the gather that it would have saved: 56 -> 67 us forward at 197 tokens.)
__device__ __forceinline__ int one_entry(const ExtArgs& a, int qt, int kt, int lo, int hi) {
    const int2 q = a.q_range[qt], k = a.k_range[kt];
    int x = lo + q.x - k.y, y = lo + q.y - k.x;
    x = x < lo ? lo : x > hi ? hi : x;
    y = y < lo ? lo : y > hi ? hi : y;
    return x == y ? x : -1;
}
// Whether all pairs of 32 queries and 32 keys fall on the table's first entry (0) or on its last (1), or neither (-1).  On a long
// sequence that is most of them, and the dQ pass, which has their dS, sums them for the table's gradient.
__device__ __forceinline__ int far_end(int2 q, int2 k, int top) { return q.y - k.x <= 0 ? 0 : q.x - k.y >= top ? 1 : -1; }
// The scores' start: the bias of 16 pairs of a lane whose own code is `mine` and the others' codes lie in LDS at `codes`
__device__ __forceinline__ void gather_bias(f32x16& st, const char* codes, int half, int mine, int lo, int hi) {
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
        const i32x4 c = *reinterpret_cast<const i32x4*>(codes + (8 * jj + 4 * half) * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) st[4 * jj + e] = lds_float(bias_at(mine, c[e], lo, hi));
    }
}
// v[i] of the pairs at table addresses at[i] into a wave's own histogram.  LDS float adds take a cycle a lane, and many times
// that where lanes meet on one address: pairs at either end of the table are summed in registers (ends), and a lane whose
// neighbour's next key falls on the same entry (positions in a row) takes that sum over, so that a diagonal of four costs one
// lane's add instead of four.
__device__ __forceinline__ void add_tile(char* hist, const int (&at)[16], float (&v)[16], int base, int top, float (&ends)[2]) {
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
#pragma unroll
        for (int e = 3; e > 0; --e) {  // lane l + 1's pair (4 jj + e) joins lane l's (4 jj + e - 1)
            const int i = 4 * jj + e;
            const float from = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v[i]), 0x130, 0xf, 0xf, true));
            const int there = __builtin_amdgcn_update_dpp(-1, at[i], 0x130, 0xf, 0xf, false);
            const bool takes = there == at[i - 1];
            v[i - 1] += takes ? from : 0.f;
            const bool gone = __builtin_amdgcn_update_dpp(0, (int)takes, 0x138, 0xf, 0xf, true) != 0;
            v[i] = gone ? 0.f : v[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        ends[0] += at[i] == base ? v[i] : 0.f;
        ends[1] += at[i] == top && top != base ? v[i] : 0.f;
        if (at[i] != base && at[i] != top && v[i] != 0.f)
            __hip_atomic_fetch_add(reinterpret_cast<float*>(hist + (at[i] - base)), v[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
}

__device__ __forceinline__ long row_offset(const ExtView& v, int r, int hkv, int G, int HD) {
    const int q = (int)fdiv((uint32_t)r, v.g);
    return (long)q * v.rs + (long)(hkv * G + (r - q * G)) * HD;
}

// what a workgroup works on
struct Job {
    int b, hkv, bh, tile, split, len, rows;  // len: valid keys; rows: live rows (self attention: those before len)
};
template <bool FEW = false>
__device__ __forceinline__ Job job_of(const ExtArgs& a, int tiles, int splits) {
    Job j;
    int l = FEW ? (int)blockIdx.x : xcd_order((int)blockIdx.x, (int)gridDim.x);
    if (FEW) {
        // a stream that no other workgroup reads: a token's heads at the same time, tokens in the order of memory (512 sequences of
        // 197 keys on 12 heads: 73 us where the order below took 82)
        j.tile = 0;
        const int parts = l / a.Hkv;
        j.hkv = l - parts * a.Hkv;
        j.b = parts / splits;
        j.split = parts - j.b * splits;
    } else {
        j.split = l % splits;
        l /= splits;
        j.tile = l % tiles;
        l /= tiles;
        // heads outside, the batch inside: an XCD gets sequences of all lengths (with the batch outside the XCDs of the long ones
        // worked twice as long as the rest on a padded batch), and its head's bias table stays in its cache
        j.hkv = l / a.B;
        j.b = l - j.hkv * a.B;
    }
    j.bh = j.b * a.Hkv + j.hkv;
    int len = a.Sk;
    if (a.lens) {
        len = a.lens[j.b];
        len = len < 0 ? 0 : len > a.Sk ? a.Sk : len;
    }
    j.len = __builtin_amdgcn_readfirstlane(len);
    j.rows = a.self && j.len < a.M ? j.len : a.M;
    return j;
}

// the row's statistics; where nothing was attended to, -log2 l = -inf makes every P of the backward zero
__device__ __forceinline__ void put_stat(const ExtArgs& a, float* stat, long at, bool some, float m, float l) {
    stat[at] = some ? -m : 0.f;
    stat[a.stat_n + at] = some ? -__builtin_amdgcn_logf(l) : -kInf;
}
// The exponents of a sweep are c s + base with base = -c m, rounded: l and O are 2^off times what they are for the m that is handed
// on, off = c m + base (2^-15 at scores of 500).  Where m grows, the old sums go to the new off; at the end off is taken out, so that
// parts can be joined and the backward's P add up to 1.
__device__ __forceinline__ float sweep_end(float m, float off) { return m == -kInf ? 1.f : __builtin_amdgcn_exp2f(-off); }

template <int HD>
__device__ __forceinline__ void own_frags(bf16x8* f, const bf16* p, bool live, int half) {
    using G = AttnGeo<HD>;
#pragma unroll
    for (int s = 0; s < G::STEPS; ++s) {
#pragma unroll
        for (int k = 0; k < 8; ++k) f[s][k] = (bf16)0.f;
        if (live) f[s] = *reinterpret_cast<const bf16x8*>(p + s * 16 + half * 8);
    }
}

// ------------------------------------------------------------------------------------------------------- forward
// One sweep with a running maximum. 4 waves own 32 rows each; keys in blocks of 64 (a block of 32 doubles the barriers, one of 128 halves
// the workgroups that a CU holds). Bound by vector instructions: 117 for a tile's 8 matrix instructions at head_dim 64 (two of
// a score's seven instructions are the bias's address), two thirds of the issue slots. 128 sequences of 197 on 12 heads of 64 with a bias:
// 57 us; 32 of 577 on 16: 108; four of up to 2047 on 8 of 128: 88; 333 rows x 1025 keys, 16 heads on 4 key heads of 64, batch
// 16: 37.
template <int HD, bool BIAS>
__global__ __launch_bounds__(256, 2) void k_ext_fwd(ExtArgs a, bf16* __restrict__ out, float* __restrict__ stat, float* __restrict__ part, float* __restrict__ part_ml,
                                                 int tiles, int splits) {
    using G = AttnGeo<HD>;
    constexpr int IMG = 64 * G::ROWBYTES;
    extern __shared__ __attribute__((aligned(16))) char smem[];  // [2][K image, V image], [2][codes 1 KiB], table
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, l31 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Job j = job_of(a, tiles, splits);
    const uint32_t lds0 = lds_address(smem);
    char* codes = smem + 4 * IMG;
    const int tab = (int)lds0 + 4 * IMG + 2048;
    const int r = j.tile * 128 + wave * 32 + l31;
    const bool live = r < j.rows;
    const long orow = r < a.M ? (long)j.b * a.o.bs + row_offset(a.o, r, j.hkv, a.G, HD) : 0;

    const int nb = (j.len + 63) >> 6, per = (nb + splits - 1) / splits;
    const int kb0 = j.split * per, kb1 = kb0 + per < nb ? kb0 + per : nb;
    const bool any = j.tile * 128 < j.rows && kb0 < kb1;  // (uniform over the workgroup)

    f32x16 o[G::DT];
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
    float m = -kInf, l = 0.f, off = 0.f;

    if (any) {
        const bf16* kbase = a.k + (long)j.b * a.kv.bs + (long)j.hkv * HD;
        const bf16* vbase = a.v + (long)j.b * a.kv.bs + (long)j.hkv * HD;
        const int krs = (int)a.kv.rs;
        auto issue = [&](int kb, int buf) {
            const int valid = j.len - kb * 64 < 64 ? j.len - kb * 64 : 64;
            const uint32_t bytes = (uint32_t)(valid - 1) * (uint32_t)krs * 2u + G::ROWBYTES;
            const long at = (long)kb * 64 * krs;
            auto off = [&](int row) { return row * krs; };
            dma_block<HD, 4>(lds0 + buf * 2 * IMG, kbase + at, bytes, valid, wave, lane, off);
            dma_block<HD, 4>(lds0 + buf * 2 * IMG + IMG, vbase + at, bytes, valid, wave, lane, off);
            if (BIAS && wave == 0) dma_words(lds0 + 4 * IMG + buf * 1024, a.k_codes4 + kb * 64, lane);
        };
        issue(kb0, 0);
        if (BIAS) {  // the head's bias table
            const i32x4 rsrc = uniform_rsrc(a.tab + (long)j.hkv * a.Rp, (uint32_t)a.Rp * 4u);
            for (int p = wave; p * 256 < a.Rp; p += 4)
                lds_dma16(rsrc, (uint32_t)(p * 1024 + lane * 16), (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds0 + 4 * IMG + 2048 + p * 1024)));
        }
        bf16x8 bq[G::STEPS];
        own_frags<HD>(bq, a.q + (long)j.b * a.qv.bs + row_offset(a.qv, live ? r : 0, j.hkv, a.G, HD), live, half);
        const int qc = tab + (BIAS && live ? a.q_codes4[r] : 0), top = tab + (a.R - 1) * 4;

        for (int kb = kb0; kb < kb1; ++kb) {
            const int buf = (kb - kb0) & 1;
            dma_barrier();
            if (kb + 1 < kb1) issue(kb + 1, buf ^ 1);
            if (j.tile * 128 + wave * 32 >= j.rows) continue;  // (this wave has no rows: it helps with the staging)
            const char* Ks = smem + buf * 2 * IMG;
            const char* Vs = Ks + IMG;
            const bool both = kb * 64 + 32 < j.len;  // whether the second tile has keys
            f32x16 st[2];
            float mb = m;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                if (kt == 1 && !both) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) st[1][i] = -kInf;
                    break;
                }
                if (BIAS) {
                    gather_bias(st[kt], codes + buf * 1024 + kt * 128, half, qc, tab, top);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) st[kt][i] = 0.f;
                }
#pragma unroll
                for (int s = 0; s < G::STEPS; ++s)
                    st[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(G::rows(Ks, kt * 32 + l31, s, half), bq[s], st[kt], 0, 0, 0);
                if ((kb + 1) * 64 > j.len) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (kb * 64 + kt * 32 + acc_row(i, half) >= j.len) st[kt][i] = -kInf;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) mb = fmaxf(mb, st[kt][i]);
            }
            mb = fmaxf(mb, __shfl_xor(mb, 32, 64));
            const float mx = mb == -kInf ? 0.f : mb;  // (every key so far forbidden: m counts as 0, all P are 0)
            // one multiply-add a score, but for a bias of, say, -1e9 over a whole row: its product leaves nothing of the scores
            const bool large = BIAS && !__all(fabsf(mx) < 65536.f);
            const float base = large ? 0.f : -mx * a.c;
            if (__any(mb > m)) {
                const float now = large ? 0.f : fmaf(mx, a.c, base), alpha = __builtin_amdgcn_exp2f(fmaf(m - mx, a.c, now - off));
                off = now;
                l *= alpha;
#pragma unroll
                for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
                m = mb;
            }
            if (large) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) st[kt][i] -= mx;
            }
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                if (kt == 1 && !both) break;
                float part_l = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    st[kt][i] = __builtin_amdgcn_exp2f(fmaf(st[kt][i], a.c, base));
                    part_l += st[kt][i];
                }
                l += part_l;
#pragma unroll
                for (int blk = 0; blk < 2; ++blk) {
                    const bf16x8 p = acc_to_a(st[kt], blk);
#pragma unroll
                    for (int dt = 0; dt < G::DT; ++dt)
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(G::cols(Vs, kt * 32 + blk * 16, dt * 32, lane), p, o[dt], 0, 0, 0);
                }
            }
        }
    }
    const float end = sweep_end(m, off);
    l = (l + __shfl_xor(l, 32, 64)) * end;
    if (splits > 1) {
        if (r < a.M) {
            const long at = ((long)j.bh * splits + j.split) * a.M + r;
#pragma unroll
            for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    f32x4 t;
#pragma unroll
                    for (int e = 0; e < 4; ++e) t[e] = o[dt][4 * jj + e] * end;
                    *reinterpret_cast<f32x4*>(part + at * HD + dt * 32 + 8 * jj + 4 * half) = t;
                }
            if (half == 0) {
                part_ml[2 * at] = m;
                part_ml[2 * at + 1] = l;
            }
        }
        return;
    }
    const float inv = l > 0.f || l != l ? end / l : 0.f;
    if (stat && half == 0 && r < a.Mp) put_stat(a, stat, (long)j.bh * a.Mp + r, live && (l > 0.f || l != l), m, l);
    if (r < a.M) {
#pragma unroll
        for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
                bf16x4 t;
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = (bf16)(live ? o[dt][4 * jj + e] * inv : 0.f);
                *reinterpret_cast<bf16x4*>(out + orow + dt * 32 + 8 * jj + 4 * half) = t;
            }
    }
}

// Few rows (at most one tile of 32 for a key head: single tokens).  The four waves of a workgroup share the rows and take
// every fourth tile of 32 keys each, through an LDS ring of their own (no barrier until the join): the kernel is a stream over
// K and V, 16 to 64 KiB of it in flight per workgroup, and bound by memory: 4 sequences of 65536 keys, 8 key heads of 128, four rows
// each: 169 us, 6.4 TB/s (with the kernel above, whose waves would have one tile of rows for four: 193); 512 of 197 on 12 heads
// of 64: 64 us, 4.8 TB/s (80 there, and the backward 275 for the 139 of its counterpart).
template <int HD, bool STREAM>
__global__ __launch_bounds__(256, 2) void k_ext_fwd_few(ExtArgs a, bf16* __restrict__ out, float* __restrict__ stat,
                                                     float* __restrict__ part, float* __restrict__ part_ml, int splits) {
    using G = AttnGeo<HD>;
    constexpr int TIMG = 32 * G::ROWBYTES, STAGE = 2 * TIMG, RPP = 1024 / G::ROWBYTES, NP = 32 / RPP;
    extern __shared__ __attribute__((aligned(16))) char smem[];  // [4 waves][2 stages][K tile, V tile], then [4][32][2] floats
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, l31 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Job j = job_of<true>(a, 1, splits);
    char* ring = smem + wave * 2 * STAGE;
    const uint32_t ring_lds = lds_address(ring);
    const bool live = l31 < a.M;
    const int nt = (j.len + 31) >> 5, per = (nt + splits - 1) / splits;
    const int t0 = j.split * per, t1 = t0 + per < nt ? t0 + per : nt;
    const bf16* kbase = a.k + (long)j.b * a.kv.bs + (long)j.hkv * HD;
    const bf16* vbase = a.v + (long)j.b * a.kv.bs + (long)j.hkv * HD;
    const int krs = (int)a.kv.rs;

    auto issue = [&](int t, int buf) {
        const int valid = j.len - t * 32 < 32 ? j.len - t * 32 : 32;
        const long at = (long)t * 32 * krs;
        dma_tile<HD, STREAM>(ring_lds + buf * STAGE, kbase + at, krs, valid, lane);
        dma_tile<HD, STREAM>(ring_lds + buf * STAGE + TIMG, vbase + at, krs, valid, lane);
    };
    f32x16 o[G::DT];
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
    float m = -kInf, l = 0.f, off = 0.f;
    int buf = 0;
    if (t0 + wave < t1) issue(t0 + wave, 0);  // (before the rows: 8.5 us for 9.5 on 8 x 12 heads of up to 1500 keys)
    bf16x8 bq[G::STEPS];
    own_frags<HD>(bq, a.q + (long)j.b * a.qv.bs + row_offset(a.qv, live ? l31 : 0, j.hkv, a.G, HD), live, half);
#pragma unroll
    for (int s = 0; s < G::STEPS; ++s) asm volatile("" : "+v"(bq[s])::"memory");  // the rows are here: only DMA is counted below
    for (int t = t0 + wave; t < t1; t += 4, buf ^= 1) {
        // the reads of the other stage (last tile) are done before it is written again
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (t + 4 < t1) {
            issue(t + 4, buf ^ 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NP) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        const char* Ks = ring + buf * STAGE;
        const char* Vs = Ks + TIMG;
        f32x16 st;
#pragma unroll
        for (int i = 0; i < 16; ++i) st[i] = 0.f;
#pragma unroll
        for (int s = 0; s < G::STEPS; ++s)
            st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(G::rows(Ks, l31, s, half), bq[s], st, 0, 0, 0);
        if ((t + 1) * 32 > j.len) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (t * 32 + acc_row(i, half) >= j.len) st[i] = -kInf;
        }
        float mb = m;
#pragma unroll
        for (int i = 0; i < 16; ++i) mb = fmaxf(mb, st[i]);
        mb = fmaxf(mb, __shfl_xor(mb, 32, 64));
        const float mx = mb == -kInf ? 0.f : mb, base = -mx * a.c;  // (every score so far -inf: m counts as 0, all P are 0)
        if (__any(mb > m)) {
            const float now = fmaf(mx, a.c, base), alpha = __builtin_amdgcn_exp2f(fmaf(m - mx, a.c, now - off));
            off = now;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
            m = mb;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            st[i] = __builtin_amdgcn_exp2f(fmaf(st[i], a.c, base));
            l += st[i];
        }
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            const bf16x8 p = acc_to_a(st, blk);
#pragma unroll
            for (int dt = 0; dt < G::DT; ++dt)
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(G::cols(Vs, blk * 16, dt * 32, lane), p, o[dt], 0, 0, 0);
        }
    }
    const float end = sweep_end(m, off);
    l = (l + __shfl_xor(l, 32, 64)) * end;
    // the waves' (m, l, O) through LDS, over their rings
    float* ml = reinterpret_cast<float*>(smem + 8 * STAGE);
    if (half == 0) {
        ml[(wave * 32 + l31) * 2] = m;
        ml[(wave * 32 + l31) * 2 + 1] = l;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    float* acc = reinterpret_cast<float*>(ring);  // [32 rows][HD]: a wave's two stages are at least that large
    static_assert(2 * STAGE >= 32 * HD * 4, "the join uses the ring");
    if (live) {
#pragma unroll
        for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
                f32x4 t;
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = o[dt][4 * jj + e] * end;
                *reinterpret_cast<f32x4*>(acc + l31 * HD + dt * 32 + 8 * jj + 4 * half) = t;
            }
    }
    __syncthreads();
    for (int i = tid; i < a.M * (HD / 4); i += 256) {
        const int r = i / (HD / 4), d = i % (HD / 4) * 4;
        float mx = -kInf, sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) mx = fmaxf(mx, ml[(w * 32 + r) * 2]);
        f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float mw = ml[(w * 32 + r) * 2], f = mw == -kInf ? 0.f : __builtin_amdgcn_exp2f((mw - mx) * a.c);
            sum += ml[(w * 32 + r) * 2 + 1] * f;
            const f32x4 u = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(smem + w * 2 * STAGE) + r * HD + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] += u[e] * f;
        }
        if (splits > 1) {
            const long at = ((long)j.bh * splits + j.split) * a.M + r;
            *reinterpret_cast<f32x4*>(part + at * HD + d) = t;
            if (d == 0) {
                part_ml[2 * at] = mx;
                part_ml[2 * at + 1] = sum;
            }
        } else {
            const bool some = sum > 0.f || sum != sum;
            const float inv = some ? 1.f / sum : 0.f;
            bf16x4 w4;
#pragma unroll
            for (int e = 0; e < 4; ++e) w4[e] = (bf16)(t[e] * inv);
            *reinterpret_cast<bf16x4*>(out + (long)j.b * a.o.bs + row_offset(a.o, r, j.hkv, a.G, HD) + d) = w4;
            if (stat && d == 0) put_stat(a, stat, (long)j.bh * a.Mp + r, some, mx, sum);
        }
    }
    if (stat && splits == 1)
        for (int r = a.M + tid; r < a.Mp; r += 256) put_stat(a, stat, (long)j.bh * a.Mp + r, false, 0.f, 0.f);
}

// (m, l, O) of the splits -> out (and stat).  HD / 4 lanes take a row's channels.  MANY: a workgroup has one row, and 1024 / HD
// groups of lanes every so many-th split, added in order; the loads of a group's splits are independent (one thread over 16
// splits took 11 us where this takes 5).  Else every group has a row of its own (6924 rows of two splits: 4 us for 9).
template <int HD, bool MANY>
__global__ __launch_bounds__(256) void k_ext_join(ExtArgs a, const float* __restrict__ part, const float* __restrict__ part_ml,
                                                  bf16* __restrict__ out, float* __restrict__ stat, int splits, int rows_of_all) {
    constexpr int W = HD / 4, NG = 256 / W;
    __shared__ __attribute__((aligned(16))) float red[MANY ? NG : 1][HD + 4];
    const int d = (int)(threadIdx.x % W) * 4, g = (int)threadIdx.x / W;
    const int row = MANY ? (int)blockIdx.x : (int)blockIdx.x * NG + g;
    if (!MANY && row >= rows_of_all) return;
    const int bh = row / a.M, r = row - bh * a.M;
    const int b = bh / a.Hkv, hkv = bh - b * a.Hkv;
    const long at0 = (long)bh * splits * a.M + r;
    if (stat && r == a.M - 1)  // padding rows of the statistics
        for (int i = a.M + (MANY ? (int)threadIdx.x : d >> 2); i < a.Mp; i += MANY ? 256 : W)
            put_stat(a, stat, (long)bh * a.Mp + i, false, 0.f, 0.f);
    float mx = -kInf, sum = 0.f;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) mx = fmaxf(mx, part_ml[2 * (at0 + (long)s * a.M)]);
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = MANY ? g : 0; s < splits; s += MANY ? NG : 1) {
        const long at = at0 + (long)s * a.M;
        const float ms = part_ml[2 * at], f = ms == -kInf ? 0.f : __builtin_amdgcn_exp2f((ms - mx) * a.c);
        sum += part_ml[2 * at + 1] * f;
        const f32x4 u = *reinterpret_cast<const f32x4*>(part + at * HD + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] += u[e] * f;
    }
    if (MANY) {
        *reinterpret_cast<f32x4*>(&red[g][d]) = t;
        if (d == 0) red[g][HD] = sum;
        __syncthreads();
        if (g > 0) return;
#pragma unroll
        for (int i = 1; i < NG; ++i) {
            const f32x4 u = *reinterpret_cast<const f32x4*>(&red[i][d]);
            if (i < splits) {
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] += u[e];
            }
        }
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < NG; ++i) sum += red[i][HD];
    }
    int rows = a.M;
    if (a.self && a.lens) {
        const int len = a.lens[b] < 0 ? 0 : a.lens[b];
        rows = len < rows ? len : rows;
    }
    const bool some = (sum > 0.f || sum != sum) && r < rows;
    const float inv = some ? 1.f / sum : 0.f;
    const long o = (long)b * a.o.bs + row_offset(a.o, r, hkv, a.G, HD) + d;
    bf16x4 w4;
#pragma unroll
    for (int e = 0; e < 4; ++e) w4[e] = (bf16)(some ? t[e] * inv : 0.f);
    *reinterpret_cast<bf16x4*>(out + o) = w4;
    if (stat && d == 0) put_stat(a, stat, (long)bh * a.Mp + r, some, mx, sum);
}

// ------------------------------------------------------------------------------------------------------- backward
// dst rows <- scale * (sum of the splits' fp32 partials, in order), or, for dead rows, what the partials hold: zeros.  One launch
// for dQ, dK and dV, as far as they are split (a launch each: 12 us for 5 on one sequence of 577).
struct SumJob {
    const float* part;
    bf16* dst;
    ExtView v;
    int G, rows, splits;
    float scale;
};
struct SumJobs {
    SumJob job[3];
};
template <int HD>
__global__ __launch_bounds__(256) void k_ext_sum(SumJobs jobs, int Hkv, long BH) {
    const SumJob& w = jobs.job[blockIdx.y];
    const float* part = w.part;
    const int rows = w.rows, splits = w.splits;
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= BH * rows * (HD / 4)) return;
    const int d = (int)(i % (HD / 4)) * 4;
    const long row = i / (HD / 4);
    const int bh = (int)(row / rows), r = (int)(row - (long)bh * rows);
    const int b = bh / Hkv, hkv = bh - b * Hkv;
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < splits; ++s) {
        const f32x4 u = *reinterpret_cast<const f32x4*>(part + (((long)bh * splits + s) * rows + r) * HD + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] += u[e];
    }
    bf16x4 w4;
#pragma unroll
    for (int e = 0; e < 4; ++e) w4[e] = (bf16)(t[e] * w.scale);
    *reinterpret_cast<bf16x4*>(w.dst + (long)b * w.v.bs + row_offset(w.v, r, hkv, w.G, HD) + d) = w4;
}

// a lane's accumulator columns: dst[d] for d = dt*32 + 8*jj + 4*half + e
template <int HD>
__device__ __forceinline__ void store_acc(const f32x16* t, bf16* dst, float scale, int half) {
    using G = AttnGeo<HD>;
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
            bf16x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = (bf16)(t[dt][4 * jj + e] * scale);
            *reinterpret_cast<bf16x4*>(dst + dt * 32 + 8 * jj + 4 * half) = w;
        }
}
template <int HD>
__device__ __forceinline__ void store_acc32(const f32x16* t, float* dst, int half) {
    using G = AttnGeo<HD>;
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
            f32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = t[dt][4 * jj + e];
            *reinterpret_cast<f32x4*>(dst + dt * 32 + 8 * jj + 4 * half) = w;
        }
}

// The same 32 rows (lane = row) through a tile image in LDS, so that a store writes whole rows, 16 B a lane: 8-byte pieces of 32
// rows at a time cost the pass over single queries a quarter of its time.  One wave, its own image.
template <int HD, bool STREAM>
__device__ __forceinline__ void store_tile(const f32x16* t, char* img, bf16* dst, int rs, int valid, float scale, int lane) {
    using G = AttnGeo<HD>;
    constexpr int RPP = 1024 / G::ROWBYTES, NP = 32 / RPP;
    const int half = lane >> 5, l31 = lane & 31;
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
            bf16x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = (bf16)(t[dt][4 * jj + e] * scale);
            *reinterpret_cast<bf16x4*>(img + G::swz(l31, dt * 4 + jj) + half * 8) = w;
        }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int row = p * RPP + lane / G::NCH;
        const int x = ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)) & (G::NCH - 1);
        const u32x4 v = *reinterpret_cast<const u32x4*>(img + p * 1024 + lane * 16);
        bf16* to = dst + (long)row * rs + ((lane % G::NCH) ^ x) * 8;
        if (row < valid && STREAM) st_stream(to, v);
        else if (row < valid) *reinterpret_cast<u32x4*>(to) = v;
    }
}

// Row owner: dQ, and D for what follows. Bound as the forward is, with half the vector instructions' slots and half of LDS in
// use and three waves a SIMD: 75 us, 123, 108 and 40 at the sizes given there. dO . O carries the rounding of P and O to bf16,
// and the sum of a row's P (dP - dO . O) is exactly what it is off by (as a row's P add up to 1): added, D is good to 32 bits,
// which the fp32 gradient of the bias table needs; that sum costs an add a score, keeping O's remainder in the forward cost it
// a quarter of its time. Where all keys are in one block dS is corrected too: with few keys P (dP - D) is a small difference.
// Without a bias and with more keys O is small against V, its rounding against dP, and nothing is added. A softmax over one key
// is constant, so with len = 1 dS is zero, and is set so (as a difference of two rounded numbers it would not be).
// FAR: `ends` [2][B Hkv][tiles of 32 rows] gets the sums of dS over the pairs of far_end's tiles, which the bias gradient's own passes
// then leave out: sum P (dP - dO . O) - delta sum P, for 18 more vector instructions a tile.  Four sequences of up to 2047 with a
// table of 257: this pass 104 -> 108 us, the sums over the batch 118 -> 41 and the entries 20 -> 13.
template <int HD, bool BIAS, bool ONE /* all keys in one block of 64 */, bool FAR>
__global__ __launch_bounds__(256, 2) void k_ext_bwd_q(ExtArgs a, const bf16* __restrict__ out, const bf16* __restrict__ dout, const float* __restrict__ stat,
                                                   float* __restrict__ dsum, float* __restrict__ ends, bf16* __restrict__ dq,
                                                   float* __restrict__ part, int tiles, int splits) {
    using G = AttnGeo<HD>;
    constexpr int IMG = 64 * G::ROWBYTES;
    extern __shared__ __attribute__((aligned(16))) char smem[];  // [2][K, V], [2][codes 1 KiB], table
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, l31 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Job j = job_of(a, tiles, splits);
    const uint32_t lds0 = lds_address(smem);
    char* codes = smem + 4 * IMG;
    const int tab = (int)lds0 + 4 * IMG + 2048;
    const int r = j.tile * 128 + wave * 32 + l31;
    const bool live = r < j.rows;
    const int nb = (j.len + 63) >> 6, per = (nb + splits - 1) / splits;
    const int kb0 = j.split * per, kb1 = kb0 + per < nb ? kb0 + per : nb;
    const bool any = j.tile * 128 < j.rows && kb0 < kb1;

    f32x16 acc[G::DT];
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;
    const bf16* kbase = a.k + (long)j.b * a.kv.bs + (long)j.hkv * HD;
    const bf16* vbase = a.v + (long)j.b * a.kv.bs + (long)j.hkv * HD;
    const int krs = (int)a.kv.rs;
    auto issue = [&](int kb, int buf) {
        const int valid = j.len - kb * 64 < 64 ? j.len - kb * 64 : 64;
        const uint32_t bytes = (uint32_t)(valid - 1) * (uint32_t)krs * 2u + G::ROWBYTES;
        const long at = (long)kb * 64 * krs;
        auto off = [&](int row) { return row * krs; };
        dma_block<HD, 4>(lds0 + buf * 2 * IMG, kbase + at, bytes, valid, wave, lane, off);
        dma_block<HD, 4>(lds0 + buf * 2 * IMG + IMG, vbase + at, bytes, valid, wave, lane, off);
        if (BIAS && wave == 0) dma_words(lds0 + 4 * IMG + buf * 1024, a.k_codes4 + kb * 64, lane);
    };
    if (any) issue(kb0, 0);
    if (BIAS && any) {
        const i32x4 rsrc = uniform_rsrc(a.tab + (long)j.hkv * a.Rp, (uint32_t)a.Rp * 4u);
        for (int p = wave; p * 256 < a.Rp; p += 4)
            lds_dma16(rsrc, (uint32_t)(p * 1024 + lane * 16), (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds0 + 4 * IMG + 2048 + p * 1024)));
    }
    // own rows, and D from them
    bf16x8 qf[G::STEPS], gf[G::STEPS];
    float d = 0.f, delta = 0.f;
    {
        const long ro = row_offset(a.o, live ? r : 0, j.hkv, a.G, HD) + (long)j.b * a.o.bs;
        own_frags<HD>(qf, a.q + (long)j.b * a.qv.bs + row_offset(a.qv, live ? r : 0, j.hkv, a.G, HD), live, half);
        own_frags<HD>(gf, dout + ro, live, half);
        bf16x8 of[G::STEPS];
        own_frags<HD>(of, out + ro, live, half);
#pragma unroll
        for (int s = 0; s < G::STEPS; ++s)
#pragma unroll
            for (int k = 0; k < 8; ++k) d += (float)of[s][k] * (float)gf[s][k];
        d += __shfl_xor(d, 32, 64);
    }
    const float mq = live ? stat[(long)j.bh * a.Mp + r] : 0.f;
    const float lq = live && j.len > 1 ? stat[a.stat_n + (long)j.bh * a.Mp + r] : -kInf;
    const int qc = tab + (BIAS && live ? a.q_codes4[r] : 0), top = tab + (a.R - 1) * 4;

    uint64_t low = 0, high = 0;  // far_end of the 64 tiles of keys at hand
    float end_off[2] = {0.f, 0.f}, end_p[2] = {0.f, 0.f};
    if (any) {
        for (int kb = kb0; kb < kb1; ++kb) {
            const int buf = (kb - kb0) & 1;
            dma_barrier();
            if (kb + 1 < kb1) issue(kb + 1, buf ^ 1);
            if (j.tile * 128 + wave * 32 >= j.rows) continue;
            if (FAR && (kb & 31) == 0) {
                const int kt = kb * 2 + lane;
                const int end = kt * 32 < a.Sk ? far_end(a.q_range[j.tile * 4 + wave], a.k_range[kt], (a.R - 1) * 4) : -1;
                low = __ballot(end == 0);
                high = __ballot(end == 1);
            }
            const char* Ks = smem + buf * 2 * IMG;
            const char* Vs = Ks + IMG;
            const bool both = kb * 64 + 32 < j.len;
            f32x16 ds[ONE ? 2 : 1], pr[ONE ? 2 : 1];
            auto product = [&](const f32x16& x, int kt) {
#pragma unroll
                for (int blk = 0; blk < 2; ++blk) {
                    const bf16x8 d8 = acc_to_a(x, blk);
#pragma unroll
                    for (int dt = 0; dt < G::DT; ++dt)
                        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(G::cols(Ks, kt * 32 + blk * 16, dt * 32, lane), d8, acc[dt], 0, 0, 0);
                }
            };
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                if (!ONE && kt == 1 && !both) break;
                f32x16 sc, dp;
                if (BIAS) gather_bias(sc, codes + buf * 1024 + kt * 128, half, qc, tab, top);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (!BIAS) sc[i] = mq;
                    dp[i] = -d;
                }
#pragma unroll
                for (int s = 0; s < G::STEPS; ++s) {
                    sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(G::rows(Ks, kt * 32 + l31, s, half), qf[s], sc, 0, 0, 0);
                    dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(G::rows(Vs, kt * 32 + l31, s, half), gf[s], dp, 0, 0, 0);
                }
                if ((kb + 1) * 64 > j.len) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (kb * 64 + kt * 32 + acc_row(i, half) >= j.len) sc[i] = -kInf;
                }
                float off = 0.f, sum_p = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(BIAS ? sc[i] + mq : sc[i], a.c, lq));
                    if (FAR) sum_p += p;
                    if (ONE) pr[kt][i] = p;
                    dp[i] *= p;
                    if (BIAS || ONE) off += dp[i];
                }
                delta += off;
                if (FAR) {
                    const int bit = (kb & 31) * 2 + kt;
                    const bool is_low = low >> bit & 1, is_high = high >> bit & 1;
                    end_off[0] += is_low ? off : 0.f;
                    end_p[0] += is_low ? sum_p : 0.f;
                    end_off[1] += is_high ? off : 0.f;
                    end_p[1] += is_high ? sum_p : 0.f;
                }
                if (ONE) ds[kt] = dp;
                else product(dp, kt);
            }
            if (ONE) {
                const float off = delta + __shfl_xor(delta, 32, 64);
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) ds[kt][i] = fmaf(-off, pr[kt][i], ds[kt][i]);
                    product(ds[kt], kt);
                }
            }
        }
    }
    delta += __shfl_xor(delta, 32, 64);
    if (FAR) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float s = row_sum(fmaf(-delta, end_p[e], end_off[e]));
            if (lane == 0) ends[((long)e * a.B * a.Hkv + j.bh) * tiles * 4 + j.tile * 4 + wave] = s;
        }
    }
    // -D of this split's keys: the first split has dO . O too, the sum over the splits is made where there is more than one
    if (half == 0 && r < a.Mp) dsum[((long)j.split * a.B * a.Hkv + j.bh) * a.Mp + r] = live ? -(delta + (j.split == 0 ? d : 0.f)) : 0.f;
    if (r >= a.M) return;
    if (splits > 1) store_acc32<HD>(acc, part + (((long)j.bh * splits + j.split) * a.M + r) * HD, half);
    else store_acc<HD>(acc, dq + (long)j.b * a.dqv.bs + row_offset(a.dqv, r, j.hkv, a.G, HD), a.scale, half);
}

// Few rows (at most 32 for a key head: an attention pooling head's query): everything in one pass over K and V.  A wave takes
// every fourth tile of 32 keys through a ring of its own, makes the tile's scores in both orientations (two small products; the
// pass is bound by the stream of K, V, dK and dV), stores dK and dV of its keys and keeps its part of dQ, which the four
// waves join at the end.  512 sequences of 197 keys, 12 heads of 64: 139 us, 4.5 TB/s; row owner and key owner took 275.
template <int HD, bool STREAM>
__global__ __launch_bounds__(256, HD > 64 ? 1 : 2) void k_ext_bwd_few(ExtArgs a, const bf16* __restrict__ out, const bf16* __restrict__ dout, const float* __restrict__ stat,
                                                        bf16* __restrict__ dq, bf16* __restrict__ dk, bf16* __restrict__ dv,
                                                        float* __restrict__ part, int splits) {
    using G = AttnGeo<HD>;
    constexpr int TIMG = 32 * G::ROWBYTES, STAGE = 2 * TIMG, NP = TIMG / 1024;
    extern __shared__ __attribute__((aligned(16))) char smem[];  // [4 waves][2 stages][K, V], Q image, dO image, [3][32] floats
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, l31 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Job j = job_of<true>(a, 1, splits);
    char* ring = smem + wave * 2 * STAGE;
    const uint32_t ring_lds = lds_address(ring);
    char* Qs = smem + 8 * STAGE;
    char* Gs = Qs + TIMG;
    float* st = reinterpret_cast<float*>(Gs + TIMG);  // -m, -log2 l, -D
    const bool live = l31 < a.M;
    const int nt = (j.len + 31) >> 5, all = (a.Sk + 31) >> 5, per = (all + splits - 1) / splits;
    const int t0 = j.split * per, t1 = t0 + per < all ? t0 + per : all;
    const bf16* kbase = a.k + (long)j.b * a.kv.bs + (long)j.hkv * HD;
    const bf16* vbase = a.v + (long)j.b * a.kv.bs + (long)j.hkv * HD;
    const int krs = (int)a.kv.rs;
    auto issue = [&](int t, int buf) {
        const int valid = j.len - t * 32 < 32 ? j.len - t * 32 : 32;
        const long at = (long)t * 32 * krs;
        dma_tile<HD, STREAM>(ring_lds + buf * STAGE, kbase + at, krs, valid, lane);
        dma_tile<HD, STREAM>(ring_lds + buf * STAGE + TIMG, vbase + at, krs, valid, lane);
    };
    if (t0 + wave < t1 && t0 + wave < nt) issue(t0 + wave, 0);
    // the rows as operands of both orientations (lane = row), their images for the products over rows, and D
    bf16x8 qf[G::STEPS], gf[G::STEPS];
    float mq, lq, d = 0.f;
    {
        const long ro = row_offset(a.o, live ? l31 : 0, j.hkv, a.G, HD) + (long)j.b * a.o.bs;
        own_frags<HD>(qf, a.q + (long)j.b * a.qv.bs + row_offset(a.qv, live ? l31 : 0, j.hkv, a.G, HD), live, half);
        own_frags<HD>(gf, dout + ro, live, half);
        bf16x8 of[G::STEPS];
        own_frags<HD>(of, out + ro, live, half);
#pragma unroll
        for (int s = 0; s < G::STEPS; ++s)
#pragma unroll
            for (int k = 0; k < 8; ++k) d -= (float)of[s][k] * (float)gf[s][k];
        d += __shfl_xor(d, 32, 64);
        const long sr = (long)j.bh * a.Mp + l31;
        mq = live ? stat[sr] : 0.f;
        lq = live ? stat[a.stat_n + sr] : -kInf;
        if (wave == 0) {
#pragma unroll
            for (int s = 0; s < G::STEPS; ++s) {
                *reinterpret_cast<bf16x8*>(Qs + G::swz(l31, 2 * s + half)) = qf[s];
                *reinterpret_cast<bf16x8*>(Gs + G::swz(l31, 2 * s + half)) = gf[s];
            }
            if (half == 0) {
                st[l31] = mq;
                st[32 + l31] = lq;
                st[64 + l31] = d;
            }
        }
        if (j.len <= 1) lq = -kInf;  // (dS of one key is zero; P for dV comes from the other orientation)
    }
    __syncthreads();
    f32x16 acc[G::DT];
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;
    int buf = 0;
    for (int t = t0 + wave; t < t1; t += 4) {
        const int key = t * 32 + l31;
        const long at = (long)j.b * a.dkv.bs + (long)t * 32 * a.dkv.rs + (long)j.hkv * HD;
        const int rows = a.Sk - t * 32 < 32 ? a.Sk - t * 32 : 32;
        if (t >= nt) {  // past the valid keys: zeros
            const u32x4 z = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const int row = p * (32 / NP) + lane / G::NCH;
                if (row < rows) {
                    *reinterpret_cast<u32x4*>(dk + at + (long)row * a.dkv.rs + (lane % G::NCH) * 8) = z;
                    *reinterpret_cast<u32x4*>(dv + at + (long)row * a.dkv.rs + (lane % G::NCH) * 8) = z;
                }
            }
            continue;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the other stage has been read
        if (t + 4 < t1 && t + 4 < nt) {
            issue(t + 4, buf ^ 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NP) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        const char* Ks = ring + buf * STAGE;
        const char* Vs = Ks + TIMG;
        buf ^= 1;  // (this tile's stage is buf ^ 1 from here)
        bf16x8 kf[G::STEPS], vf[G::STEPS];
#pragma unroll
        for (int s = 0; s < G::STEPS; ++s) {
            kf[s] = G::rows(Ks, l31, s, half);
            vf[s] = G::rows(Vs, l31, s, half);
        }
        {  // lane = row, registers = keys: dQ
            f32x16 sc, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                sc[i] = mq;
                dp[i] = d;
            }
#pragma unroll
            for (int s = 0; s < G::STEPS; ++s) {
                sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[s], qf[s], sc, 0, 0, 0);
                dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[s], gf[s], dp, 0, 0, 0);
            }
            if ((t + 1) * 32 > j.len) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (t * 32 + acc_row(i, half) >= j.len) sc[i] = -kInf;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) dp[i] *= __builtin_amdgcn_exp2f(fmaf(sc[i], a.c, lq));
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
                const bf16x8 ds = acc_to_a(dp, blk);
#pragma unroll
                for (int dt = 0; dt < G::DT; ++dt)
                    acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(G::cols(Ks, blk * 16, dt * 32, lane), ds, acc[dt], 0, 0, 0);
            }
        }
        {  // lane = key, registers = rows: dK, dV
            f32x16 sc, dp, o[G::DT];
            f32x4 lr[4];
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
                const f32x4 mr = *reinterpret_cast<const f32x4*>(st + 8 * jj + 4 * half);
                lr[jj] = *reinterpret_cast<const f32x4*>(st + 32 + 8 * jj + 4 * half);
                const f32x4 dr = *reinterpret_cast<const f32x4*>(st + 64 + 8 * jj + 4 * half);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[4 * jj + e] = mr[e];
                    dp[4 * jj + e] = dr[e];
                }
            }
#pragma unroll
            for (int s = 0; s < G::STEPS; ++s) {
                sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf[s], kf[s], sc, 0, 0, 0);
                dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(gf[s], vf[s], dp, 0, 0, 0);
            }
            const bool key_live = key < j.len;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                sc[i] = key_live ? __builtin_amdgcn_exp2f(fmaf(sc[i], a.c, lr[i >> 2][i & 3])) : 0.f;
                dp[i] = key_live && j.len > 1 ? dp[i] * sc[i] : 0.f;
            }
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const char* img = g ? Qs : Gs;
#pragma unroll
                for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
#pragma unroll
                for (int blk = 0; blk < 2; ++blk) {
                    const bf16x8 x = acc_to_a(g ? dp : sc, blk);
#pragma unroll
                    for (int dt = 0; dt < G::DT; ++dt)
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(G::cols(img, blk * 16, dt * 32, lane), x, o[dt], 0, 0, 0);
                }
                // (the tile's own images are free: its rows are in registers, its columns were read for dQ)
                store_tile<HD, STREAM>(o, ring + (buf ^ 1) * STAGE + (g ? 0 : TIMG), (g ? dk : dv) + at, (int)a.dkv.rs, rows, g ? a.scale : 1.f, lane);
            }
        }
    }
    // the waves' parts of dQ through their rings
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    float* mine = reinterpret_cast<float*>(ring);
    static_assert(2 * STAGE >= 32 * HD * 4, "the join uses the ring");
    store_acc32<HD>(acc, mine + l31 * HD, half);
    __syncthreads();
    for (int i = tid; i < a.M * (HD / 4); i += 256) {
        const int r = i / (HD / 4), c = i % (HD / 4) * 4;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const f32x4 u = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(smem + w * 2 * STAGE) + r * HD + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += u[e];
        }
        if (splits > 1) {
            *reinterpret_cast<f32x4*>(part + (((long)j.bh * splits + j.split) * a.M + r) * HD + c) = s;
        } else {
            bf16x4 w4;
#pragma unroll
            for (int e = 0; e < 4; ++e) w4[e] = (bf16)(s[e] * a.scale);
            *reinterpret_cast<bf16x4*>(dq + (long)j.b * a.dqv.bs + row_offset(a.dqv, r, j.hkv, a.G, HD) + c) = w4;
        }
    }
}

// dsum[0] <- the sum of the splits' parts of -D, in order
__global__ __launch_bounds__(256) void k_ext_dsum(float* __restrict__ dsum, long n, int splits) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float s = dsum[i];
    for (int k = 1; k < splits; ++k) s += dsum[k * n + i];
    dsum[i] = s;
}

// dS summed over a part of the batch, for 128 queries x 128 keys of a head a workgroup (a wave: 32 queries, four tiles of 32
// keys).  The bias of the block and the sums stay in registers while the batch streams through, so a pair costs two
// multiply-adds and an exponential per sequence; written in register order, [tile][4][64 lanes] x 4 floats.  Its bound is what the
// blocks move from L2, 64 KiB for 128 x 128 pairs of head_dim 64, at 6 to 7 TB/s: 60 us, 139 and 39 at the sizes given at the
// forward.  Blocks of 256 x 256 with the bias gathered for every sequence (no registers left for it) took 85 and 248, a second buffer
// for K and V 64 and 149.
template <int HD>
__global__ __launch_bounds__(256, 2) void k_rel_dbias(ExtArgs a, const bf16* __restrict__ dout, const float* __restrict__ stat,
                                                      const float* __restrict__ dsum, float* __restrict__ dense, RelBlocks w) {
    using G = AttnGeo<HD>;
    constexpr int IMG = 128 * G::ROWBYTES;  // as two blocks of 64 rows
    extern __shared__ __attribute__((aligned(16))) char smem[];  // K, V of one sequence; before that the table
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, l31 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int l = xcd_order((int)blockIdx.x, (int)gridDim.x);
    const int kb = l % w.kblocks;
    l /= w.kblocks;
    const int qb = l % w.qblocks + w.q0;
    l /= w.qblocks;
    const int hl = l % w.heads, h = hl + w.h0, ch = l / w.heads;
    const int per = (a.B + w.chunks - 1) / w.chunks, b0 = ch * per, b1 = b0 + per < a.B ? b0 + per : a.B;
    const uint32_t lds0 = lds_address(smem);
    const int q = qb * 128 + wave * 32 + l31, krs = (int)a.kv.rs;
    if (w.ends) {  // nothing to do where the dQ pass has all sixteen tiles (lanes 0 to 15 look at one each)
        const int qt = qb * 4 + (lane & 3), kt = kb * 4 + (lane >> 2 & 3);
        if (__all(qt * 32 >= a.Sk || kt * 32 >= a.Sk || far_end(a.q_range[qt], a.k_range[kt], (a.R - 1) * 4) >= 0)) return;
    }

    // the block's bias (minus nothing yet): the table through LDS
    f32x16 bias[4], acc[4];
    {
        const i32x4 rsrc = uniform_rsrc(a.tab + (long)h * a.Rp, (uint32_t)a.Rp * 4u);
        for (int p = wave; p * 256 < a.Rp; p += 4)
            lds_dma16(rsrc, (uint32_t)(p * 1024 + lane * 16), (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds0 + p * 1024)));
        const int qc = (int)lds0 + a.q_codes4[q], top = (int)lds0 + (a.R - 1) * 4;
        dma_barrier();
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
                const i32x4 kc = *reinterpret_cast<const i32x4*>(a.k_codes4 + kb * 128 + kt * 32 + 8 * jj + 4 * half);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    bias[kt][4 * jj + e] = lds_float(bias_at(qc, kc[e], (int)lds0, top));
                    acc[kt][4 * jj + e] = 0.f;
                }
            }
        dma_barrier();
    }
    for (int b = b0; b < b1; ++b) {
        int len = a.Sk;
        if (a.lens) {
            len = a.lens[b];
            len = __builtin_amdgcn_readfirstlane(len < 0 ? 0 : len > a.Sk ? a.Sk : len);
        }
        if (len <= 1 || kb * 128 >= len || qb * 128 >= len) continue;  // (one key: dS is zero)
        const long kvb = (long)b * a.kv.bs + (long)h * HD + (long)kb * 128 * krs;
        auto off = [&](int row) { return row * krs; };
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int left = len - kb * 128 - s * 64, valid = left < 0 ? 0 : left < 64 ? left : 64;
            const uint32_t bytes = valid ? (uint32_t)(valid - 1) * (uint32_t)krs * 2u + G::ROWBYTES : 0u;
            dma_block<HD, 4>(lds0 + s * (IMG / 2), a.k + kvb + (long)s * 64 * krs, bytes, valid, wave, lane, off);
            dma_block<HD, 4>(lds0 + IMG + s * (IMG / 2), a.v + kvb + (long)s * 64 * krs, bytes, valid, wave, lane, off);
        }
        const bool live = q < len;
        bf16x8 qf[G::STEPS], gf[G::STEPS];
        own_frags<HD>(qf, a.q + (long)b * a.qv.bs + (long)(live ? q : 0) * a.qv.rs + (long)h * HD, live, half);
        own_frags<HD>(gf, dout + (long)b * a.o.bs + (long)(live ? q : 0) * a.o.rs + (long)h * HD, live, half);
        const long sr = ((long)b * a.Hkv + h) * a.Mp + (live ? q : 0);
        const float mq = live ? stat[sr] : 0.f, lq = live ? stat[a.stat_n + sr] : -kInf, d = live ? dsum[sr] : 0.f;
        dma_barrier();
        if (qb * 128 + wave * 32 < len) {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                if (kb * 128 + kt * 32 < len) {
                    const char* Ks = smem + (kt >> 1) * (IMG / 2);
                    const char* Vs = Ks + IMG;
                    f32x16 sc, dp;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        sc[i] = bias[kt][i];
                        dp[i] = d;
                    }
#pragma unroll
                    for (int s = 0; s < G::STEPS; ++s) {
                        sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(G::rows(Ks, (kt & 1) * 32 + l31, s, half), qf[s], sc, 0, 0, 0);
                        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(G::rows(Vs, (kt & 1) * 32 + l31, s, half), gf[s], dp, 0, 0, 0);
                    }
                    if (kb * 128 + kt * 32 + 32 > len) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (kb * 128 + kt * 32 + acc_row(i, half) >= len) sc[i] = -kInf;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[kt][i] = fmaf(__builtin_amdgcn_exp2f(fmaf(sc[i] + mq, a.c, lq)), dp[i], acc[kt][i]);
                }
            }
        }
        dma_barrier();
    }
    const int nkt = w.kblocks * 4;
    const long row = ((long)ch * w.heads + hl) * (w.qblocks * 4) + (qb - w.q0) * 4 + wave;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
        if (kb * 128 + kt * 32 >= a.Sk || qb * 128 + wave * 32 >= a.Sk) break;  // (tiles that are not read)
        float* dst = dense + (row * nkt + kb * 4 + kt) * 1024 + lane * 4;
        if (w.ends && far_end(a.q_range[qb * 4 + wave], a.k_range[kb * 4 + kt], (a.R - 1) * 4) >= 0) continue;
        if (one_entry(a, qb * 4 + wave, kb * 4 + kt, 0, (a.R - 1) * 4) >= 0) {  // one number
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) s += acc[kt][i];
            s = row_sum(s);
            if (lane == 0) dst[0] = s;
            continue;
        }
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
            f32x4 t;
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = acc[kt][4 * jj + e];
            *reinterpret_cast<f32x4*>(dst + jj * 256) = t;
        }
    }
}

// The pairs' sums by entry (9, 20 and 13 us there, most of it the LDS adds and the histograms' clearing): a workgroup takes a
// tile row (32 queries) of a head and one of `parts` shares of its key tiles, each wave with a histogram of its own.  Shares are
// neighbouring tiles (20 us where tiles in turn took 21), but tiles in turn where the dQ pass has the far ones (13 for 18:
// what is left lies together).
__global__ __launch_bounds__(256) void k_rel_entries(ExtArgs a, const float* __restrict__ dense, float* __restrict__ slab, RelBlocks w,
                                                     int parts) {
    extern __shared__ __attribute__((aligned(16))) char smem[];  // [4][Rp] floats
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, l31 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int part = (int)blockIdx.x % parts, rest = (int)blockIdx.x / parts, nqt = w.qblocks * 4, nkt = w.kblocks * 4;
    const int qt = rest % nqt, hl = rest / nqt;
    float* hist = reinterpret_cast<float*>(smem) + (long)wave * a.Rp;
    const int base = (int)lds_address(hist), top = base + (a.R - 1) * 4;
    for (int i = lane * 4; i < a.Rp; i += 256) *reinterpret_cast<f32x4*>(hist + i) = f32x4{0.f, 0.f, 0.f, 0.f};  // (Rp: a multiple of 4)
    const int q = (w.q0 * 4 + qt) * 32 + l31;
    const int qc = base + a.q_codes4[q];
    const int live_t = (a.Sk + 31) / 32, per = (live_t + parts - 1) / parts, last = w.ends || (part + 1) * per > live_t ? live_t : (part + 1) * per;
    const int t1 = w.q0 * 4 + qt < live_t ? last : 0, step_t = w.ends ? 4 * parts : 4;
    float ends[2] = {0.f, 0.f};
    if (w.ends && part == 0 && wave == 0)
#pragma unroll 4
        for (int b = lane; b < a.B; b += 64)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                ends[e] += w.ends[(((long)e * a.B + b) * a.Hkv + hl + w.h0) * (w.kblocks * 4) + w.q0 * 4 + qt];
    for (int kt = (w.ends ? part * 4 : part * per) + wave; kt < t1; kt += step_t) {
        if (w.ends && far_end(a.q_range[w.q0 * 4 + qt], a.k_range[kt], (a.R - 1) * 4) >= 0) continue;
        const float* src = dense + (((long)hl * nqt + qt) * nkt + kt) * 1024 + lane * 4;
        const long step = (long)w.heads * nqt * nkt * 1024;
        const int one = one_entry(a, w.q0 * 4 + qt, kt, base, top);
        if (one >= 0) {
            if (lane == 0) {
                float s = 0.f;
                for (int ch = 0; ch < w.chunks; ++ch) s += src[ch * step];
                hist[(one - base) >> 2] += s;
            }
            continue;
        }
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0.f;
#pragma unroll 4
        for (int ch = 0; ch < w.chunks; ++ch) {
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
                const f32x4 t = *reinterpret_cast<const f32x4*>(src + ch * step + jj * 256);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * jj + e] += t[e];
            }
        }
        int at[16];
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
            const i32x4 kc = *reinterpret_cast<const i32x4*>(a.k_codes4 + kt * 32 + 8 * jj + 4 * half);
#pragma unroll
            for (int e = 0; e < 4; ++e) at[4 * jj + e] = bias_at(qc, kc[e], base, top);
        }
        add_tile(reinterpret_cast<char*>(hist), at, v, base, top, ends);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        ends[i] = row_sum(ends[i]);
        if (lane == 0) hist[i * (a.R - 1)] += ends[i];
    }
    __syncthreads();
    float* dst = slab + ((long)(hl + w.h0) * w.slab_rows + (long)(w.q0 * 4 + qt) * parts + part) * a.Rp;
    const float* all = reinterpret_cast<const float*>(smem);
    for (int i = tid * 4; i < a.Rp; i += 1024) {
        f32x4 s = *reinterpret_cast<const f32x4*>(all + i);
#pragma unroll
        for (int w4 = 1; w4 < 4; ++w4) {
            const f32x4 u = *reinterpret_cast<const f32x4*>(all + w4 * a.Rp + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += u[e];
        }
        *reinterpret_cast<f32x4*>(dst + i) = s;
    }
}

// Key owner: dK and dV of 128 keys a workgroup; the rows of all G heads stream through. Four products
// a tile for the row owner's three, and a row's numbers (-m, -log2 l, -D, code) come from LDS for every register: 92 us, 160, 170 and 54 at the
// sizes given at the forward, LDS and vector instructions half busy each. -D and the exponent by a matrix instruction with ones
// instead: 99 and 67; the exponent as one number with a branch for large maxima: 101.
template <int HD, bool BIAS>
__global__ __launch_bounds__(256, HD > 64 ? 1 : BIAS ? 3 : 2) void k_ext_bwd_kv(ExtArgs a, const bf16* __restrict__ dout, const float* __restrict__ stat,
                                                    const float* __restrict__ dsum, bf16* __restrict__ dk, bf16* __restrict__ dv,
                                                    float* __restrict__ part_k, float* __restrict__ part_v, int tiles, int splits) {
    using G = AttnGeo<HD>;
    constexpr int IMG = 64 * G::ROWBYTES;
    extern __shared__ __attribute__((aligned(16))) char smem[];  // [2][Q, dO], [2][-log2 l, -D, codes, -m: 1 KiB each], table
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, l31 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Job j = job_of(a, tiles, splits);
    const uint32_t lds0 = lds_address(smem);
    char* stat_s = smem + 4 * IMG;
    const int tab = (int)lds0 + 4 * IMG + 8192;
    const int key = j.tile * 128 + wave * 32 + l31;
    const bool live = key < j.len;
    const int nb = (j.rows + 63) >> 6, per = (nb + splits - 1) / splits;
    const int rb0 = j.split * per, rb1 = rb0 + per < nb ? rb0 + per : nb;
    const bool any = j.tile * 128 < j.len && rb0 < rb1;

    f32x16 ak[G::DT], av[G::DT];
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            ak[dt][i] = 0.f;
            av[dt][i] = 0.f;
        }
    if (any) {
        const bf16* qb = a.q + (long)j.b * a.qv.bs + (long)j.hkv * a.G * HD;
        const bf16* gb = dout + (long)j.b * a.o.bs + (long)j.hkv * a.G * HD;
        const int qrs = (int)a.qv.rs, grs = (int)a.o.rs;
        const float* mrow = stat + (long)j.bh * a.Mp;
        const float* lrow = mrow + a.stat_n;
        const float* drow = dsum + (long)j.bh * a.Mp;
        auto issue = [&](int rb, int buf) {
            const int valid = j.rows - rb * 64 < 64 ? j.rows - rb * 64 : 64;
            const int q0 = (int)fdiv((uint32_t)(rb * 64), a.qv.g), last = (int)fdiv((uint32_t)(rb * 64 + valid - 1), a.qv.g);
            const uint32_t span = (uint32_t)(last - q0), width = (uint32_t)(a.G * HD * 2);
            auto qoff = [&](int row) {
                const int q = (int)fdiv((uint32_t)(rb * 64 + row), a.qv.g);
                return (q - q0) * qrs + (rb * 64 + row - q * a.G) * HD;
            };
            auto goff = [&](int row) {
                const int q = (int)fdiv((uint32_t)(rb * 64 + row), a.qv.g);
                return (q - q0) * grs + (rb * 64 + row - q * a.G) * HD;
            };
            dma_block<HD, 4>(lds0 + buf * 2 * IMG, qb + (long)q0 * qrs, span * (uint32_t)qrs * 2u + width, valid, wave, lane, qoff);
            dma_block<HD, 4>(lds0 + buf * 2 * IMG + IMG, gb + (long)q0 * grs, span * (uint32_t)grs * 2u + width, valid, wave, lane, goff);
            const uint32_t st = lds0 + 4 * IMG + buf * 4096;
            if (wave == 0) dma_words(st, lrow + rb * 64, lane);
            if (wave == 1) dma_words(st + 1024, drow + rb * 64, lane);
            if (BIAS && wave == 2) dma_words(st + 2048, a.q_codes4 + rb * 64, lane);
            if (wave == 3) dma_words(st + 3 * 1024, mrow + rb * 64, lane);
        };
        issue(rb0, 0);
        if (BIAS) {
            const i32x4 rsrc = uniform_rsrc(a.tab + (long)j.hkv * a.Rp, (uint32_t)a.Rp * 4u);
            for (int p = wave; p * 256 < a.Rp; p += 4)
                lds_dma16(rsrc, (uint32_t)(p * 1024 + lane * 16), (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds0 + 4 * IMG + 8192 + p * 1024)));
        }
        bf16x8 kf[G::STEPS], vf[G::STEPS];
        const long ko = (long)j.b * a.kv.bs + (long)(live ? key : 0) * a.kv.rs + (long)j.hkv * HD;
        own_frags<HD>(kf, a.k + ko, live, half);
        own_frags<HD>(vf, a.v + ko, live, half);
        const int kc = (BIAS && live ? a.k_codes4[key] : 0) - tab, top = tab + (a.R - 1) * 4;

        for (int rb = rb0; rb < rb1; ++rb) {
            const int buf = (rb - rb0) & 1;
            dma_barrier();
            if (rb + 1 < rb1) issue(rb + 1, buf ^ 1);
            // (a wave without keys helps with the staging.  head_dim 128 has one wave a SIMD and lives on the overlap of its two
            // row tiles: 170 us on four sequences of up to 2047, 203 us with this branch or the next one)
            if (HD <= 64 && j.tile * 128 + wave * 32 >= j.len) continue;
            const char* Qs = smem + buf * 2 * IMG;
            const char* Gs = Qs + IMG;
            const char* st = stat_s + buf * 4096;
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) {
                if (HD <= 64 && rt == 1 && rb * 64 + 32 >= j.rows) break;
                f32x16 sc, dp;
                // With a bias -m is needed after the products.  Held through them, -m and -log2 l cost a SIMD its third wave at head_dim
                // 64 (103 us at 128 x 197 x 12 heads where read late 91); at 128, with one wave, late reads wait (196 us for 171).
                constexpr bool LATE = BIAS && HD <= 64;
                f32x4 lr[4], mr[4];
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    const int w = (rt * 32 + 8 * jj + 4 * half) * 4;
                    if (!LATE) {
                        lr[jj] = *reinterpret_cast<const f32x4*>(st + w);
                        mr[jj] = *reinterpret_cast<const f32x4*>(st + 3 * 1024 + w);
                    }
                    const f32x4 dr = *reinterpret_cast<const f32x4*>(st + 1024 + w);
                    i32x4 qc = {0, 0, 0, 0};
                    if (BIAS) qc = *reinterpret_cast<const i32x4*>(st + 2048 + w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[4 * jj + e] = BIAS ? lds_float(bias_at(qc[e], kc, tab, top)) : mr[jj][e];
                        dp[4 * jj + e] = dr[e];
                    }
                }
#pragma unroll
                for (int s = 0; s < G::STEPS; ++s) {
                    sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(G::rows(Qs, rt * 32 + l31, s, half), kf[s], sc, 0, 0, 0);
                    dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(G::rows(Gs, rt * 32 + l31, s, half), vf[s], dp, 0, 0, 0);
                }
                // (no mask: a dead key is a lane of its own whose results are not stored; rows past the end have -log2 l = -inf)
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    const int w = (rt * 32 + 8 * jj + 4 * half) * 4;
                    if (LATE) {
                        asm volatile("" ::: "memory");
                        mr[jj] = *reinterpret_cast<const f32x4*>(st + 3 * 1024 + w);
                        lr[jj] = *reinterpret_cast<const f32x4*>(st + w);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = 4 * jj + e;
                        const float p = __builtin_amdgcn_exp2f(fmaf(BIAS ? sc[i] + mr[jj][e] : sc[i], a.c, lr[jj][e]));
                        sc[i] = p;
                        dp[i] *= p;
                    }
                }
#pragma unroll
                for (int blk = 0; blk < 2; ++blk) {
                    const bf16x8 p = acc_to_a(sc, blk), ds = acc_to_a(dp, blk);
#pragma unroll
                    for (int dt = 0; dt < G::DT; ++dt) {
                        av[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(G::cols(Gs, rt * 32 + blk * 16, dt * 32, lane), p, av[dt], 0, 0, 0);
                        ak[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(G::cols(Qs, rt * 32 + blk * 16, dt * 32, lane), ds, ak[dt], 0, 0, 0);
                    }
                }
            }
        }
    }
    if (key >= a.Sk) return;
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (!live) av[dt][i] = 0.f;
            if (!live || j.len <= 1) ak[dt][i] = 0.f;
        }
    if (splits > 1) {
        const long at = (((long)j.bh * splits + j.split) * a.Sk + key) * HD;
        store_acc32<HD>(ak, part_k + at, half);
        store_acc32<HD>(av, part_v + at, half);
    } else {
        const long at = (long)j.b * a.dkv.bs + (long)key * a.dkv.rs + (long)j.hkv * HD;
        store_acc<HD>(ak, dk + at, a.scale, half);
        store_acc<HD>(av, dv + at, 1.f, half);
    }
}

// ------------------------------------------------------------------------------------------------------- bias tables
// tab[h][r] = table[bucket_of[r]][h] * sqrt(hd) (the scores are scaled after the bias is added), zero where the entry names no
// bucket; byte offsets of the position codes, padded with the last one to a multiple of 128 (what is past the end then falls
// on an entry that its neighbours use).  Offsets, their differences and an LDS address fit 32 bits where the codes are below
// kCodeReach in magnitude.  What matters of a difference is its place in a table of at most 4096 entries, so larger codes move in:
// those above the reach keep their distances from the lowest of them, kCodeSpan of them, and are kCodeGap from the others where they
// are further; those below likewise.  Left are pairs past the span on one side: where a query and a key are, the table is NaN,
// and so is every result: a limit without a sync, but not without a word.  (Every workgroup looks at all codes by itself: 2.3 ->
// 3.1 us on 50 tokens, 4.7 -> 5.0 on 197 to 2047.)
constexpr long kCodeReach = 1L << 27, kCodeSpan = (1L << 27) - (1L << 18), kCodeGap = 2 * kExtMaxEntries;
static_assert(8 * (kCodeReach + kCodeSpan + 2 * kCodeGap) + 163840 < 1L << 31, "byte offsets' differences and an LDS address fit 32 bits");
struct CodeEdges {
    long low, high;  // the largest code below -kCodeReach, the smallest from kCodeReach on
};
__device__ __forceinline__ long code_at(const void* codes, bool wide, int i) {
    return wide ? static_cast<const long*>(codes)[i] : (long)static_cast<const int*>(codes)[i];
}
// how far past the span of its side a code is, or less than 0
__device__ __forceinline__ long past_span(long c, const CodeEdges& e) {
    return c >= kCodeReach ? c - e.high - kCodeSpan : c < -kCodeReach ? e.low - c - kCodeSpan : -1;
}
__device__ __forceinline__ int moved_in(long c, const CodeEdges& e) {
    if (c >= -kCodeReach && c < kCodeReach) return (int)c;
    const bool up = c >= kCodeReach;
    const long gap = up ? e.high - kCodeReach : -kCodeReach - e.low;  // (from the reach to the first)
    const long out = kCodeReach + min(gap, kCodeGap) + (past_span(c, e) >= 0 ? kCodeSpan + kCodeGap : up ? c - e.high : e.low - c);
    return (int)(up ? out : -out);
}
// whether a code is past the reach (256 threads, four loads of each axis in flight)
template <typename Q, typename K>
__device__ __forceinline__ bool codes_past_reach(const void* q_codes, const void* k_codes, int S) {
    bool past = false;
    for (int i0 = (int)threadIdx.x; i0 < S; i0 += 1024) {
        Q q[4];
        K k[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int i = i0 + 256 * n < S ? i0 + 256 * n : i0;
            q[n] = static_cast<const Q*>(q_codes)[i];
            k[n] = static_cast<const K*>(k_codes)[i];
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) past |= q[n] < -kCodeReach || q[n] >= kCodeReach || k[n] < -kCodeReach || k[n] >= kCodeReach;
    }
    return past;
}
// the edges of both sides, and whether a query's and a key's code are both past the span of one
__device__ __forceinline__ bool code_edges(const void* q_codes, bool q_wide, const void* k_codes, bool k_wide, int S, CodeEdges& e) {
    __shared__ long edge[2][4];
    __shared__ int past[4];
    const int wave = threadIdx.x >> 6;
    e = {-__LONG_MAX__ - 1, __LONG_MAX__};
    for (int i = (int)threadIdx.x; i < 2 * S; i += 256) {
        const long c = i < S ? code_at(q_codes, q_wide, i) : code_at(k_codes, k_wide, i - S);
        if (c >= kCodeReach) e.high = min(e.high, c);
        if (c < -kCodeReach) e.low = max(e.low, c);
    }
    for (int n = 1; n < 64; n *= 2) {
        e.high = min(e.high, __shfl_xor(e.high, n, 64));
        e.low = max(e.low, __shfl_xor(e.low, n, 64));
    }
    edge[0][wave] = e.low;  // (all lanes the same)
    edge[1][wave] = e.high;
    __syncthreads();
    for (int n = 0; n < 4; ++n) {
        e.low = max(e.low, edge[0][n]);
        e.high = min(e.high, edge[1][n]);
    }
    int bits = 0;  // 1, 2: a query's above, below; 4, 8: a key's
    for (int i = (int)threadIdx.x; i < 2 * S; i += 256) {
        const long c = i < S ? code_at(q_codes, q_wide, i) : code_at(k_codes, k_wide, i - S);
        if (past_span(c, e) >= 0) bits |= (c > 0 ? 1 : 2) << (i < S ? 0 : 2);
    }
    for (int n = 1; n < 64; n *= 2) bits |= __shfl_xor(bits, n, 64);
    past[wave] = bits;
    __syncthreads();
    bits = past[0] | past[1] | past[2] | past[3];
    return ((bits & 5) == 5) || ((bits & 10) == 10);
}
__global__ __launch_bounds__(256) void k_bias_tables(const float* __restrict__ table, const int* __restrict__ bucket_of,
                                                     const void* __restrict__ q_codes, bool q_wide, const void* __restrict__ k_codes, bool k_wide,
                                                     float* __restrict__ tab, int* __restrict__ codes /* q4 [Sp], k4 [Sp], ranges of 32 */, int R,
                                                     int Rp, int NB, int H, int S, int Sp, float inv_scale, int tab_blocks) {
    const bool is_tab = (int)blockIdx.x < tab_blocks;
    // what this thread writes, loaded before the codes are looked at: an entry, or a code
    const uint32_t i = blockIdx.x * 256 + threadIdx.x, h = i / (uint32_t)Rp, r = i - h * (uint32_t)Rp;
    const int w = ((int)blockIdx.x - tab_blocks) * 256 + (int)threadIdx.x, at = w < Sp ? w : w - Sp;  // (2 Sp: a multiple of 256)
    float v = 0.f;
    long code = 0;
    if (!is_tab) {
        code = code_at(w < Sp ? q_codes : k_codes, w < Sp ? q_wide : k_wide, at < S ? at : S - 1);
    } else if (h < (uint32_t)H) {
        const int n = r < (uint32_t)R ? bucket_of[r] : -1;
        v = n >= 0 && n < NB ? finite_bias(table[(long)n * H + h]) : 0.f;
    }
    const bool past = !q_wide && !k_wide ? codes_past_reach<int, int>(q_codes, k_codes, S)
                      : !q_wide          ? codes_past_reach<int, long>(q_codes, k_codes, S)
                      : !k_wide          ? codes_past_reach<long, int>(q_codes, k_codes, S)
                                         : codes_past_reach<long, long>(q_codes, k_codes, S);
    CodeEdges edges{};
    bool too_far = false;
    if (__syncthreads_or(past)) too_far = code_edges(q_codes, q_wide, k_codes, k_wide, S, edges);
    if (is_tab) {
        if (h < (uint32_t)H) tab[i] = too_far ? __builtin_nanf("") : v * inv_scale;
        return;
    }
    const int c = moved_in(code, edges) * 4;
    codes[w] = c;
    int lo = c, hi = c;
#pragma unroll
    for (int e = 1; e < 32; e *= 2) {
        const int l = __shfl_xor(lo, e, 64), u = __shfl_xor(hi, e, 64);
        lo = l < lo ? l : lo;
        hi = u > hi ? u : hi;
    }
    if ((threadIdx.x & 31) == 0) reinterpret_cast<int2*>(codes + 2L * Sp)[w >> 5] = {lo, hi};
}

// sums[h][r] = sum of the slab rows [H][rows][Rp] of head h: 64 entries a workgroup, each of its four waves every fourth row
__global__ __launch_bounds__(256) void k_bias_slab(const float* __restrict__ slab, float* __restrict__ sums, int Rp, int rows) {
    __shared__ float red[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = blockIdx.x * 64 + lane, h = blockIdx.y;
    float s = 0.f;
    if (r < Rp) {
#pragma unroll 8
        for (int i = wave; i < rows; i += 4) s += slab[((long)h * rows + i) * Rp + r];
    }
    red[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && r < Rp) sums[(long)h * Rp + r] = red[0][lane] + red[1][lane] + red[2][lane] + red[3][lane];
}

// dtable[n][h] = sum over the entries r of bucket n: a lane per bucket, a workgroup takes 64 buckets, its 16 waves every 16th 64
// entries.  Entries lie a lane each and go round by readlane; 64 whose buckets are all in other workgroups (on a grid nearly
// all: there an entry is a bucket) are passed over.  Any number of entries may share a bucket, in any order.
// `rows` rows of sums a head.
__global__ __launch_bounds__(1024) void k_bias_buckets(const float* __restrict__ slab, int rows, const int* __restrict__ bucket_of,
                                                      float* __restrict__ dtable, int R, int Rp, int NB, int H) {
    __shared__ float red[16][64];
    const int h = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = blockIdx.x * 64 + lane;
    float s = 0.f;
    for (int r0 = wave * 64; r0 < R; r0 += 1024) {
        const int r = r0 + lane, of = r < R ? bucket_of[r] - (int)blockIdx.x * 64 : -1;
        if (!__any(of >= 0 && of < 64)) continue;
        float v = 0.f;
        if (r < R) {
#pragma unroll 8
            for (int i = 0; i < rows; ++i) v += slab[((long)h * rows + i) * Rp + r];
        }
#pragma unroll 8
        for (int e = 0; e < 64; ++e) {
            const float x = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), e));
            s += __builtin_amdgcn_readlane(of, e) == lane ? x : 0.f;
        }
    }
    red[wave][lane] = s;
    __syncthreads();
    if (wave > 0 || n >= NB) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i][lane];
    dtable[(long)n * H + h] = s;
}

template <typename K>
void allow_lds(K kern, size_t bytes) {
    if (bytes <= 65536) return;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != hipSuccess) throw std::runtime_error(std::string("attention: ") + hipGetErrorString(e));  // (an exception of the call)
}

// Whether the passes over few rows take and leave K and V with the non-temporal hint: where K and V are more than the 256 MB that
// lie in front of the memory.  310 MB: forward 74 -> 62 us, backward 147 -> 139; 1 GB: 185 -> 169; but 123 MB: backward 45 -> 55,
// 110 MB: forward 24 -> 25.
bool streams_past_caches(const ExtArgs& a, int hd) { return 4L * a.B * a.Sk * a.Hkv * hd >= 256L << 20; }

size_t table_bytes(const ExtArgs& a) { return a.tab ? (size_t)((a.Rp + 255) & ~255) * 4 : 0; }

template <int HD>
void fwd(const ExtArgs& a, const ExtPlan& p, void* out, float* stat, float* part, float* part_ml, hipStream_t s) {
    const unsigned grid = (unsigned)((long)a.B * a.Hkv * p.tiles * p.splits);
    if (p.few) {
        const size_t lds = (size_t)16 * 32 * HD * 2 + 4 * 32 * 2 * sizeof(float);
        const auto kern = streams_past_caches(a, HD) ? &k_ext_fwd_few<HD, true> : &k_ext_fwd_few<HD, false>;
        allow_lds(kern, lds);
        hipLaunchKernelGGL(kern, dim3(grid), dim3(256), lds, s, a, (bf16*)out, stat, part, part_ml, p.splits);
    } else {
        const size_t lds = (size_t)4 * 64 * HD * 2 + (a.tab ? 2048 : 0) + table_bytes(a);
#define PDT_EXT_FWD(BIAS)                                                                                               \
    allow_lds(&k_ext_fwd<HD, BIAS>, lds);                                                                              \
    hipLaunchKernelGGL((k_ext_fwd<HD, BIAS>), dim3(grid), dim3(256), lds, s, a, (bf16*)out, stat, part, part_ml, p.tiles, p.splits);
        if (a.tab) {
            PDT_EXT_FWD(true)
        } else {
            PDT_EXT_FWD(false)
        }
#undef PDT_EXT_FWD
    }
    if (p.splits > 1) {
        const int rows = (int)((long)a.B * a.Hkv * a.M), ng = 1024 / HD;  // (a launch that is split has at most 256 tiles of 128 rows)
        if (p.splits > 4)
            hipLaunchKernelGGL((k_ext_join<HD, true>), dim3((unsigned)rows), dim3(256), 0, s, a, (const float*)part, (const float*)part_ml,
                               (bf16*)out, stat, p.splits, rows);
        else
            hipLaunchKernelGGL((k_ext_join<HD, false>), dim3((unsigned)((rows + ng - 1) / ng)), dim3(256), 0, s, a, (const float*)part,
                               (const float*)part_ml, (bf16*)out, stat, p.splits, rows);
    }
}

template <int HD>
void bwd(const ExtArgs& a, const ExtBwd& w, hipStream_t s) {
    const ExtPlan &pq = w.q, &pk = w.kv;
    const dim3 gq((unsigned)((long)a.B * a.Hkv * pq.tiles * pq.splits)), gk((unsigned)((long)a.B * a.Hkv * pk.tiles * pk.splits));
    if (pq.few) {
        const size_t lds = (size_t)(16 + 2) * 32 * HD * 2 + 3 * 32 * sizeof(float);
        const auto kern = streams_past_caches(a, HD) ? &k_ext_bwd_few<HD, true> : &k_ext_bwd_few<HD, false>;
        allow_lds(kern, lds);
        hipLaunchKernelGGL(kern, gq, dim3(256), lds, s, a, (const bf16*)w.out, (const bf16*)w.dout, w.stat, (bf16*)w.dq, (bf16*)w.dk, (bf16*)w.dv, w.part_q, pq.splits);
    } else {
        const size_t lq = (size_t)4 * 64 * HD * 2 + (a.tab ? 2048 : 0) + table_bytes(a);
        const size_t lk = (size_t)4 * 64 * HD * 2 + 8192 + table_bytes(a);
        const long n = a.stat_n;
#define PDT_EXT_BWD_Q(BIAS, ONE, FAR)                                                                                    \
    allow_lds(&k_ext_bwd_q<HD, BIAS, ONE, FAR>, lq);                                                                     \
    hipLaunchKernelGGL((k_ext_bwd_q<HD, BIAS, ONE, FAR>), gq, dim3(256), lq, s, a, (const bf16*)w.out, (const bf16*)w.dout, w.stat, \
                       w.dsum, w.ends, (bf16*)w.dq, w.part_q, pq.tiles, pq.splits);
#define PDT_EXT_BWD_KV(BIAS)                                                                                              \
    allow_lds(&k_ext_bwd_kv<HD, BIAS>, lk);                                                                               \
    hipLaunchKernelGGL((k_ext_bwd_kv<HD, BIAS>), gk, dim3(256), lk, s, a, (const bf16*)w.dout, w.stat, (const float*)w.dsum, \
                       (bf16*)w.dk, (bf16*)w.dv, w.part_k, w.part_v, pk.tiles, pk.splits);
        const bool one = a.Sk <= 64;
        if (a.tab && one) {
            PDT_EXT_BWD_Q(true, true, false)
        } else if (a.tab && w.ends) {
            PDT_EXT_BWD_Q(true, false, true)
        } else if (a.tab) {
            PDT_EXT_BWD_Q(true, false, false)
        } else if (one) {
            PDT_EXT_BWD_Q(false, true, false)
        } else {
            PDT_EXT_BWD_Q(false, false, false)
        }
        if (pq.splits > 1) hipLaunchKernelGGL(k_ext_dsum, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, w.dsum, n, pq.splits);
        if (a.tab) {
            PDT_EXT_BWD_KV(true)
        } else {
            PDT_EXT_BWD_KV(false)
        }
#undef PDT_EXT_BWD_Q
#undef PDT_EXT_BWD_KV
    }
    const long BH = (long)a.B * a.Hkv;
    SumJobs jobs{};
    unsigned n = 0;
    int rows = 0;
    auto add = [&](const float* part, void* dst, const ExtView& v, int G, int m, int splits, float scale) {
        if (splits < 2) return;
        jobs.job[n++] = {part, (bf16*)dst, v, G, m, splits, scale};
        rows = m > rows ? m : rows;
    };
    add(w.part_q, w.dq, a.dqv, a.G, a.M, pq.splits, a.scale);
    add(w.part_k, w.dk, a.dkv, 1, a.Sk, pk.splits, a.scale);
    add(w.part_v, w.dv, a.dkv, 1, a.Sk, pk.splits, 1.f);
    if (n)
        hipLaunchKernelGGL((k_ext_sum<HD>), dim3((unsigned)((BH * rows * (HD / 4) + 255) / 256), n), dim3(256), 0, s, jobs, a.Hkv, BH);
}

// parts to cut `blocks` blocks of the streamed axis into, so that `groups` workgroups become about two per CU (512); a part
// keeps at least `least` blocks. Cut and joined against whole: one sequence of 577 on 12 heads, training, 100 us for 112; 64
// rows x 2000 keys on 8 heads, forward and dQ, 27 us for 72; single rows over 1500 and over 65536 keys, 11 and 190 us for 12
// and 705. 256 or 1024 workgroups instead of 512 changed none of these by 5 %. With 300 workgroups cutting lost: five sequences
// of 577, training, 144 us whole and 149 cut; single rows over 1500 keys on 24 x 12 heads 23 and 25.
int splits_for(long groups, long blocks, long least) {
    if (groups >= 256 || blocks < 2 * least) return 1;
    long s = (512 + groups - 1) / groups;
    s = s < blocks / least ? s : blocks / least;
    return (int)(s < 1 ? 1 : s > 128 ? 128 : s);
}

}  // namespace

// Up to 32 rows, one tile of a wave, the waves share them: 32 rows x 1000 keys on 40 x 12 heads of 64, training, 71 us for 116; 8 rows
// 67 for 113.  (With a bias they would want its table beside the rings.)
ExtPlan ext_plan_fwd(long BH, int M, int Sk, bool bias) {
    ExtPlan p;
    p.few = !bias && M <= 32;
    p.tiles = p.few ? 1 : (M + 127) / 128;
    p.splits = p.few ? splits_for(BH, (Sk + 31) / 32, 8) : splits_for(BH * p.tiles, (Sk + 63) / 64, 4);
    return p;
}
void ext_plan_bwd(long BH, int M, int Sk, bool bias, ExtPlan& q, ExtPlan& kv) {
    q.few = kv.few = !bias && M <= 32 && Sk > 64;  // (few keys want D exact, which is the row owner's)
    if (q.few) {  // one kernel
        q.tiles = 1;
        q.splits = splits_for(BH, (Sk + 31) / 32, 8);
        kv.tiles = kv.splits = 0;
        return;
    }
    q.tiles = (M + 127) / 128;
    q.splits = splits_for(BH * q.tiles, (Sk + 63) / 64, 4);
    kv.tiles = (Sk + 127) / 128;
    kv.splits = splits_for(BH * kv.tiles, (M + 63) / 64, 4);
}

void launch_ext_fwd(const ExtArgs& a, const ExtPlan& p, int hd, void* out, float* stat, float* part, float* part_ml,
                    hipStream_t s) {
    if (hd == 32) fwd<32>(a, p, out, stat, part, part_ml, s);
    else if (hd == 64) fwd<64>(a, p, out, stat, part, part_ml, s);
    else fwd<128>(a, p, out, stat, part, part_ml, s);
}
void launch_ext_bwd(const ExtArgs& a, const ExtBwd& w, int hd, hipStream_t s) {
    if (hd == 32) bwd<32>(a, w, s);
    else if (hd == 64) bwd<64>(a, w, s);
    else bwd<128>(a, w, s);
}
void launch_bias_tables(const float* table, const int* bucket_of, const void* q_codes, bool q_wide, const void* k_codes, bool k_wide,
                        float* tab, int* codes, int R, int Rp, int NB, int H, int S, int Sp, float inv_scale, hipStream_t s) {
    const int tab_blocks = (int)(((long)H * Rp + 255) / 256);
    hipLaunchKernelGGL(k_bias_tables, dim3((unsigned)(tab_blocks + 2L * Sp / 256)), dim3(256), 0, s, table, bucket_of, q_codes, q_wide,
                       k_codes, k_wide, tab, codes, R, Rp, NB, H, S, Sp, inv_scale, tab_blocks);
}
long ext_ends(const ExtArgs& a, const ExtPlan& q) {
    return a.tab && a.Sk > 64 && a.Sk >= a.R && q.splits == 1 ? 2L * a.B * a.Hkv * q.tiles * 4 : 0;
}
// Head groups and query blocks of a dense sum of at most 1 GiB; the batch in parts
RelPlan rel_plan(int B, int H, int S, int hd) {
    RelPlan p;
    const long blocks = (S + 127) / 128, row_block = blocks * 4 * blocks * 4 * 4096;  // bytes of a head
    const long most = 1L << 30;
    p.heads = (int)(row_block >= most ? 1 : most / row_block < H ? most / row_block : H);
    p.qblocks = (int)(row_block <= most ? blocks : most / (row_block / blocks) > 0 ? most / (row_block / blocks) : 1);
    const long groups = (long)p.heads * p.qblocks * blocks;
    // Parts of the batch: a launch runs in rounds of the 512 workgroups that the CUs hold; a round is 4 us and, per sequence of a
    // part, 4.2 us at head_dim 64, and each part's sums are written and read once at 5 TB/s.  (128 sequences of 197 on 12 heads: 10
    // parts in one round, where the 16 that fill the last of two rounds better took 58 us; 32 of 577 on 16 heads: one part, where
    // five in four rounds took 145 us, 26 of them for the sums.)
    const long part = p.heads * p.qblocks * (row_block / blocks), room = most / part, live = (S + 31) / 32;
    const double move = 2.0 * part * live * live / (16.0 * blocks * blocks) / 5e6, step = 4.2 * hd / 64;
    p.chunks = 1;
    double best = 0;
    for (int c = 1; c <= 16 && c <= B && (c == 1 || c <= room); ++c) {
        const double t = (double)((groups * c + 511) / 512) * (4 + step * ((B + c - 1) / c)) + c * move;
        if (c == 1 || t < best) {
            best = t;
            p.chunks = c;
        }
    }
    // ranges of key tiles: as many workgroups as the CUs hold at once (four each where a head has 2000 entries)
    const long rows = (long)H * blocks * 4;
    const long tiles = (S + 31) / 32;
    long q = 1024 / rows;
    q = q < (tiles + 3) / 4 ? q : (tiles + 3) / 4;
    p.parts = (int)(q < 1 ? 1 : q);
    p.rows = (int)(blocks * 4 * p.parts);
    p.dense = p.chunks * part / 4;
    return p;
}
template <int HD>
static void rel_dbias(const ExtArgs& a, const ExtBwd& x, float* dense, const RelBlocks& w, hipStream_t s) {
    const size_t tab = (size_t)((a.Rp + 255) & ~255) * 4, stage = (size_t)2 * 128 * HD * 2, lds = tab > stage ? tab : stage;
    allow_lds(&k_rel_dbias<HD>, lds);
    hipLaunchKernelGGL((k_rel_dbias<HD>), dim3((unsigned)(w.kblocks * w.qblocks * w.heads * w.chunks)), dim3(256), lds, s, a,
                       (const bf16*)x.dout, x.stat, (const float*)x.dsum, dense, w);
}
void launch_rel_bias_grad(const ExtArgs& a, const ExtBwd& x, int hd, const RelPlan& p, float* dense, float* slab, float* mid,
                          const int* bucket_of, float* dtable, int NB, hipStream_t s) {
    const int blocks = (a.Sk + 127) / 128;
    for (int h0 = 0; h0 < a.Hkv; h0 += p.heads)
        for (int q0 = 0; q0 < blocks; q0 += p.qblocks) {
            RelBlocks w;
            w.h0 = h0;
            w.heads = a.Hkv - h0 < p.heads ? a.Hkv - h0 : p.heads;
            w.q0 = q0;
            w.qblocks = blocks - q0 < p.qblocks ? blocks - q0 : p.qblocks;
            w.kblocks = blocks;
            w.chunks = p.chunks;
            w.slab_rows = p.rows;
            w.ends = x.ends;
            if (hd == 32) rel_dbias<32>(a, x, dense, w, s);
            else if (hd == 64) rel_dbias<64>(a, x, dense, w, s);
            else rel_dbias<128>(a, x, dense, w, s);
            const size_t lds = (size_t)4 * a.Rp * 4;
            allow_lds(&k_rel_entries, lds);
            hipLaunchKernelGGL(k_rel_entries, dim3((unsigned)(w.heads * w.qblocks * 4 * p.parts)), dim3(256), lds, s, a,
                               (const float*)dense, slab, w, p.parts);
        }
    // few rows of the slab are summed where they are read: 16 rows of 732 entries in 4.8 us for 9.4, but 60 of 2212 in 14.5 for 12.7
    const bool direct = p.rows <= 32;
    if (!direct) hipLaunchKernelGGL(k_bias_slab, dim3((a.Rp + 63) / 64, a.Hkv), dim3(256), 0, s, (const float*)slab, mid, a.Rp, p.rows);
    hipLaunchKernelGGL(k_bias_buckets, dim3((NB + 63) / 64, a.Hkv), dim3(1024), 0, s, (const float*)(direct ? slab : mid), direct ? p.rows : 1,
                       bucket_of, dtable, a.R, a.Rp, NB, a.Hkv);
}

}  // namespace pdt
