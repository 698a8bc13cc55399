// End of a residual block and start of the next in one pass over token-major activations [B, T, D], bf16 in and out, fp32
// statistics and parameters:
//
//   z = LN(y; pw, pb)  (or z = y)      the norm after the branch
//   u = a x + gate z                   gate [D], or [B, D] with a row for each sample
//   n = LN(u; w, b)                    the norm before the next branch, of u before it is rounded for the stream
//
// Backward, with yh / uh the normalised y / u and g = du + LN'(dn):
//   dx = a g,  dgate = sum g z,  dz = gate g,  dy = LN'(dz) (or dz),  dw = sum dn uh,  db = sum dn,  dpw = sum dz yh,  dpb = sum dz
//
// Bound by memory: forward 2 reads + 2 writes, backward 4 reads + 2 writes of 2 bytes per element.  64 x 577 rows of 1024, a gate
// for each sample: 57 us (5.3 TB/s) and 85 (5.3 TB/s) + 5 for the sums; 64 x 197 rows of 768 with the norm of the branch: 19 and
// 31 + 4.  x and y are what the backward reads again (not u): u is recomputed in fp32, so the parameter gradients see the numbers that the forward normalised,
// at no more traffic than a saved u would cost.  One wave holds a row in registers (4 channels a lane and piece, NP pieces of
// 256 channels) and walks over rows with the parameters in registers (read again for every row they were 2.7 times the
// row's own bytes) and the next row's loads in flight.  Row sums by DPP, not through LDS.  The column sums stay in registers over
// all rows a wave visits, are added over the waves in LDS and over the workgroups in a fixed order (no atomics).
#include "attn_tile.h"
#include "gated_norm.h"

namespace pdt {
namespace {

constexpr int kMaxPieces = 8;  // D <= 2048

__device__ __forceinline__ bf16x4 raw4(const bf16* p, bool in) {
    bf16x4 t = {(bf16)0.f, (bf16)0.f, (bf16)0.f, (bf16)0.f};
    if (in) t = *reinterpret_cast<const bf16x4*>(p);
    return t;
}
template <bool STREAM>
__device__ __forceinline__ void put4(bf16* p, bf16x4 v) {
    if (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<bf16x4*>(p));
    else *reinterpret_cast<bf16x4*>(p) = v;
}
__device__ __forceinline__ f32x4 par4(const float* p, bool in) {
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
    if (in) t = *reinterpret_cast<const f32x4*>(p);
    return t;
}
template <int NP, bool POST, bool STREAM>
__global__ __launch_bounds__(256, NP <= 3 ? 4 : NP == 4 ? 3 : NP < 8 ? 2 : 1) void k_gn_fwd(GatedNorm p, bf16* __restrict__ u_out, bf16* __restrict__ n_out,
                                                                  float* __restrict__ stats /* [2 or 4][M], or null */) {
    const int lane = threadIdx.x & 63, D = p.D, np4 = D >> 2;
    const long stride = (long)gridDim.x * 4;
    long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= p.M) return;
    const float inv_d = 1.f / (float)D;
    f32x4 ga[NP], w[NP], b[NP], pw[POST ? NP : 1], pb[POST ? NP : 1];
    bf16x4 xn[NP], yn[NP];
    auto fetch = [&](long r) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int c = lane + 64 * j;
            xn[j] = raw4(p.x + r * D + 4 * c, c < np4);
            yn[j] = raw4(p.y + r * D + 4 * c, c < np4);
        }
    };
    fetch(row);
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int c = lane + 64 * j;
        w[j] = par4(p.w + 4 * c, c < np4);
        b[j] = par4(p.b + 4 * c, c < np4);
        if (POST) {
            pw[j] = par4(p.pw + 4 * c, c < np4);
            pb[j] = par4(p.pb + 4 * c, c < np4);
        }
    }
    long sample = -1;
    for (; row < p.M; row += stride) {
        float x[NP][4], y[NP][4];
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[j][k] = (float)xn[j][k];
                y[j][k] = (float)yn[j][k];
            }
        if (row + stride < p.M) fetch(row + stride);
        const long own = p.per_sample ? row / p.T : 0;
        if (own != sample) {
            sample = own;
#pragma unroll
            for (int j = 0; j < NP; ++j) ga[j] = par4(p.gate + own * D + 4 * (lane + 64 * j), lane + 64 * j < np4);
        }
        float s = 0.f, q = 0.f;
        if (POST) {
#pragma unroll
            for (int j = 0; j < NP; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) s += y[j][k];
            const float mean = row_sum(s) * inv_d;
#pragma unroll
            for (int j = 0; j < NP; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float d = lane + 64 * j < np4 ? y[j][k] - mean : 0.f;
                    q += d * d;
                }
            const float rstd = rsqrtf(row_sum(q) * inv_d + p.eps);
#pragma unroll
            for (int j = 0; j < NP; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) y[j][k] = (y[j][k] - mean) * rstd * pw[j][k] + pb[j][k];
            if (stats && lane == 0) {
                stats[2 * p.M + row] = mean;
                stats[3 * p.M + row] = rstd;
            }
        }
        s = q = 0.f;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            bf16x4 o;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[j][k] = p.a * x[j][k] + ga[j][k] * y[j][k];
                s += x[j][k];
                o[k] = (bf16)x[j][k];
            }
            if (lane + 64 * j < np4) put4<STREAM>(u_out + row * D + 4 * (lane + 64 * j), o);
        }
        const float mean = row_sum(s) * inv_d;
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float d = lane + 64 * j < np4 ? x[j][k] - mean : 0.f;
                q += d * d;
            }
        const float rstd = rsqrtf(row_sum(q) * inv_d + p.eps);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            bf16x4 o;
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = (bf16)((x[j][k] - mean) * rstd * w[j][k] + b[j][k]);
            if (lane + 64 * j < np4) *reinterpret_cast<bf16x4*>(n_out + row * D + 4 * (lane + 64 * j)) = o;
        }
        if (stats && lane == 0) {
            stats[row] = mean;
            stats[p.M + row] = rstd;
        }
    }
}

// the four waves' column sums -> dst[D] (wave order); `red` [3][NP * 256]
template <int NP>
__device__ __forceinline__ void column_sum(float (&v)[NP][4], float* red, float* dst, int lane, int wave, int np4) {
    constexpr int DP = NP * 256;
    __syncthreads();
    if (wave > 0) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const f32x4 t = {v[j][0], v[j][1], v[j][2], v[j][3]};
            *reinterpret_cast<f32x4*>(red + (wave - 1) * DP + 4 * (lane + 64 * j)) = t;
        }
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            f32x4 t = {v[j][0], v[j][1], v[j][2], v[j][3]};
#pragma unroll
            for (int w = 0; w < 3; ++w) {
                const f32x4 o = *reinterpret_cast<const f32x4*>(red + w * DP + 4 * (lane + 64 * j));
#pragma unroll
                for (int k = 0; k < 4; ++k) t[k] += o[k];
            }
            if (lane + 64 * j < np4) *reinterpret_cast<f32x4*>(dst + 4 * (lane + 64 * j)) = t;
        }
    }
#pragma unroll
    for (int j = 0; j < NP; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) v[j][k] = 0.f;
}

// A unit is one of `chunks` parts of a sample's rows; a workgroup takes the units blockIdx.x, + gridDim.x, ...  The gate's sums
// leave after every unit (to gate_part + unit * gate_stride), the others at the end (slab [gridDim.x][srow]: db, dw, dpb, dpw).
template <int NP, bool POST, bool STREAM>
__global__ __launch_bounds__(256, NP <= (POST ? 3 : 4) ? 2 : 1) void k_gn_bwd(
    GatedNorm p, const bf16* __restrict__ du, const bf16* __restrict__ dn, const float* __restrict__ stats, bf16* __restrict__ dx,
    bf16* __restrict__ dy, float* __restrict__ gate_part, long gate_stride, float* __restrict__ slab, int srow, int chunks, long units) {
    constexpr int DP = NP * 256;
    extern __shared__ __attribute__((aligned(16))) float red[];  // [3][DP] for the column sums, then the parameters, [4][DP]
    f32x4* wl = reinterpret_cast<f32x4*>(red + 3 * DP);  // (in registers they left no room for a second wave; zeros past D)
    f32x4* gl = wl + DP / 4;
    f32x4* pwl = gl + DP / 4;
    f32x4* pbl = pwl + DP / 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int D = p.D, np4 = D >> 2;
    const float inv_d = 1.f / (float)D;
    float sg[NP][4], sw[NP][4], sb[NP][4], spw[POST ? NP : 1][4], spb[POST ? NP : 1][4];
    for (int c = threadIdx.x; c < DP / 4; c += 256) {
        wl[c] = par4(p.w + 4 * c, c < np4);
        if (POST) {
            pwl[c] = par4(p.pw + 4 * c, c < np4);
            pbl[c] = par4(p.pb + 4 * c, c < np4);
        }
    }
#pragma unroll
    for (int j = 0; j < NP; ++j) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            sg[j][k] = sw[j][k] = sb[j][k] = 0.f;
            if (POST) spw[j][k] = spb[j][k] = 0.f;
        }
    }
    const long rows = p.per_sample ? p.T : p.M, per = (rows + chunks - 1) / chunks;
    for (long unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const long b = unit / chunks, ch = unit - b * chunks;
        const long r0 = b * rows + ch * per, r1 = r0 + per < (b + 1) * rows ? r0 + per : (b + 1) * rows;
        const float* gate = p.gate + (p.per_sample ? b * D : 0);
        bf16x4 xn[NP], yn[NP], gn[NP], en[NP];
        f32x4 st;
        auto fetch = [&](long r) {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                const int c = lane + 64 * j;
                const bool in = c < np4;
                xn[j] = raw4(p.x + r * D + 4 * c, in);
                yn[j] = raw4(p.y + r * D + 4 * c, in);
                en[j] = raw4(dn + r * D + 4 * c, in && dn);
                gn[j] = raw4(du + r * D + 4 * c, in && du);
            }
            st[0] = stats[r];
            st[1] = stats[p.M + r];
            if (POST) {
                st[2] = stats[2 * p.M + r];
                st[3] = stats[3 * p.M + r];
            }
        };
        if (r0 + wave < r1) fetch(r0 + wave);
        for (int c = threadIdx.x; c < DP / 4; c += 256) gl[c] = par4(gate + 4 * c, c < np4);
        __syncthreads();
        for (long row = r0 + wave; row < r1; row += 4) {
            asm volatile("" ::: "memory");  // (the parameters are read here, not kept across rows)
            float x[NP][4], y[NP][4];  // uh; yh, or y
            bf16x4 e[NP], g[NP];
            const float mu = st[0], ru = st[1], my = st[2], ry = st[3];
            float s1 = 0.f, s2 = 0.f;  // sums of dn w and dn w uh
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                e[j] = en[j];
                g[j] = gn[j];
                const f32x4 ga = gl[lane + 64 * j], w = wl[lane + 64 * j];
                f32x4 pw, pb;
                if (POST) {
                    pw = pwl[lane + 64 * j];
                    pb = pbl[lane + 64 * j];
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float z = (float)yn[j][k];
                    if (POST) z = (z - my) * ry;
                    y[j][k] = z;
                    if (POST) z = z * pw[k] + pb[k];
                    x[j][k] = (p.a * (float)xn[j][k] + ga[k] * z - mu) * ru;
                    const float d = (float)en[j][k];  // (zero past the end, and so is all that follows from it)
                    sw[j][k] += d * x[j][k];
                    sb[j][k] += d;
                    const float t = d * w[k];
                    s1 += t;
                    s2 += t * x[j][k];
                }
            }
            if (row + 4 < r1) fetch(row + 4);
            s1 = row_sum(s1) * inv_d;
            s2 = row_sum(s2) * inv_d;
            asm volatile("" ::: "memory");
            float s3 = 0.f, s4 = 0.f;
            float dz[NP][4];
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                const bool in = lane + 64 * j < np4;
                const f32x4 ga = gl[lane + 64 * j], w = wl[lane + 64 * j];
                f32x4 pw, pb;
                if (POST) {
                    pw = pwl[lane + 64 * j];
                    pb = pbl[lane + 64 * j];
                }
                bf16x4 o;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float gk = in ? (float)g[j][k] + ru * ((float)e[j][k] * w[k] - s1 - x[j][k] * s2) : 0.f;
                    o[k] = (bf16)(p.a * gk);
                    sg[j][k] += gk * (POST ? y[j][k] * pw[k] + pb[k] : y[j][k]);
                    dz[j][k] = gk * ga[k];
                    if (POST) {
                        spw[j][k] += dz[j][k] * y[j][k];
                        spb[j][k] += dz[j][k];
                        const float t = dz[j][k] * pw[k];
                        s3 += t;
                        s4 += t * y[j][k];
                    }
                }
                if (in) put4<STREAM>(dx + row * D + 4 * (lane + 64 * j), o);
            }
            if (POST) {
                s3 = row_sum(s3) * inv_d;
                s4 = row_sum(s4) * inv_d;
                asm volatile("" ::: "memory");
            }
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                f32x4 pw;
                if (POST) pw = pwl[lane + 64 * j];
                bf16x4 o;
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = (bf16)(POST ? ry * (dz[j][k] * pw[k] - s3 - y[j][k] * s4) : dz[j][k]);
                if (lane + 64 * j < np4) *reinterpret_cast<bf16x4*>(dy + row * D + 4 * (lane + 64 * j)) = o;
            }
        }
        column_sum<NP>(sg, red, gate_part + unit * gate_stride, lane, wave, np4);
    }
    float* out = slab + (long)blockIdx.x * srow;
    column_sum<NP>(sb, red, out, lane, wave, np4);
    column_sum<NP>(sw, red, out + D, lane, wave, np4);
    if constexpr (POST) {
        column_sum<NP>(spb, red, out + 2 * D, lane, wave, np4);
        column_sum<NP>(spw, red, out + 3 * D, lane, wave, np4);
    }
}

// Both sums over workgroups in one launch (two took 9 us where this takes 5).  The first sum_blocks: sums[c] = sum of the slab's
// rows [rows][n], 32 columns a workgroup (8 lanes of four), each of 32 groups of lanes every 32nd row, the groups added in
// order.  The others: dgate[b][c] = sum of the sample's units, 64 columns, a wave every fourth, the four waves added in order.
__global__ __launch_bounds__(256) void k_gn_sums(const float* __restrict__ slab, float* __restrict__ sums, int rows, int n, int sum_blocks,
                                                 const float* __restrict__ part, float* __restrict__ dgate, int D, int chunks) {
    __shared__ __attribute__((aligned(16))) float red[32][32];
    if ((int)blockIdx.x < sum_blocks) {
        const int g = threadIdx.x >> 3, q = (threadIdx.x & 7) * 4, c = blockIdx.x * 32 + q;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        if (c < n) {
#pragma unroll 8
            for (int r = g; r < rows; r += 32) {
                const f32x4 t = *reinterpret_cast<const f32x4*>(slab + (long)r * n + c);
#pragma unroll
                for (int k = 0; k < 4; ++k) s[k] += t[k];
            }
        }
        *reinterpret_cast<f32x4*>(&red[g][q]) = s;
        __syncthreads();
        if (threadIdx.x < 32 && blockIdx.x * 32 + threadIdx.x < (unsigned)n) {
            float t = 0.f;
#pragma unroll
            for (int k = 0; k < 32; ++k) t += red[k][threadIdx.x];
            sums[blockIdx.x * 32 + threadIdx.x] = t;
        }
        return;
    }
    float* wave_sums = &red[0][0];  // [4][64]
    const int at = (int)blockIdx.x - sum_blocks, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, blocks = (D + 63) / 64;
    const long b = at / blocks;
    const int c = (int)(at - b * blocks) * 64 + lane;
    float s = 0.f;
    if (c < D) {
#pragma unroll 8
        for (int k = wave; k < chunks; k += 4) s += part[(b * chunks + k) * D + c];
    }
    wave_sums[wave * 64 + lane] = s;
    __syncthreads();
    if (wave == 0 && c < D) dgate[b * D + c] = wave_sums[lane] + wave_sums[64 + lane] + wave_sums[128 + lane] + wave_sums[192 + lane];
}

}  // namespace

bool gated_norm_dim_ok(long D) { return D >= 4 && D % 4 == 0 && D <= kMaxPieces * 256; }

#define PDT_GN_CASE(N, ...) case N: { constexpr int NP = N; __VA_ARGS__; } break;
#define PDT_GN_DISPATCH(D, ...)                                                                                       \
    switch (((D) + 255) / 256) {                                                                                      \
        PDT_GN_CASE(1, __VA_ARGS__) PDT_GN_CASE(2, __VA_ARGS__) PDT_GN_CASE(3, __VA_ARGS__) PDT_GN_CASE(4, __VA_ARGS__) \
        PDT_GN_CASE(5, __VA_ARGS__) PDT_GN_CASE(6, __VA_ARGS__) PDT_GN_CASE(7, __VA_ARGS__) PDT_GN_CASE(8, __VA_ARGS__) \
        default: break; /* (the binding refuses other widths) */                                                      \
    }

void launch_gated_norm_fwd(const GatedNorm& p, void* u, void* n, float* stats, hipStream_t s) {
    const long full = (p.M + 3) / 4;
    const unsigned grid = (unsigned)(full < 1024 ? full : 1024);  // (4 per CU walk over the rows)
    PDT_GN_DISPATCH(p.D, {
        const auto kern = p.pw ? (p.stream ? &k_gn_fwd<NP, true, true> : &k_gn_fwd<NP, true, false>)
                               : (p.stream ? &k_gn_fwd<NP, false, true> : &k_gn_fwd<NP, false, false>);
        hipLaunchKernelGGL(kern, dim3(grid), dim3(256), 0, s, p, (bf16*)u, (bf16*)n, stats);
    });
}

GatedNormPlan gated_norm_plan(long B, long T, long M, bool per_sample) {
    // about 512 workgroups (2 per CU) of at least 8 rows: at 1024 their partial sums were a quarter of the kernel's traffic
    GatedNormPlan q;
    const long samples = per_sample ? B : 1, rows = per_sample ? T : M;
    long c = (512 + samples - 1) / samples;
    if (c > (rows + 7) / 8) c = (rows + 7) / 8;
    if (per_sample && c > 256) c = 256;  // (k_gn_sums walks over a sample's chunks)
    q.chunks = (int)(c < 1 ? 1 : c);
    q.units = samples * q.chunks;
    q.blocks = (int)(q.units < 512 ? q.units : 512);
    return q;
}

void launch_gated_norm_bwd(const GatedNorm& p, const GatedNormPlan& q, const void* du, const void* dn, const float* stats, void* dx,
                           void* dy, float* gate_part, long gate_stride, float* slab, int srow, hipStream_t s) {
    PDT_GN_DISPATCH(p.D, {
        const size_t lds = (size_t)7 * NP * 256 * sizeof(float);
        const auto kern = p.pw ? (p.stream ? &k_gn_bwd<NP, true, true> : &k_gn_bwd<NP, true, false>)
                               : (p.stream ? &k_gn_bwd<NP, false, true> : &k_gn_bwd<NP, false, false>);
        hipLaunchKernelGGL(kern, dim3(q.blocks), dim3(256), lds, s, p, (const bf16*)du, (const bf16*)dn, stats, (bf16*)dx, (bf16*)dy,
                           gate_part, gate_stride, slab, srow, q.chunks, q.units);
    });
}
void launch_gated_norm_sums(const float* slab, float* sums, int rows, int n, const float* part, float* dgate, long B, int D, int chunks,
                            hipStream_t s) {
    const int sum_blocks = sums ? (n + 31) / 32 : 0;
    const long gate_blocks = dgate ? B * ((D + 63) / 64) : 0;
    if (sum_blocks + gate_blocks == 0) return;
    hipLaunchKernelGGL(k_gn_sums, dim3((unsigned)(sum_blocks + gate_blocks)), dim3(256), 0, s, slab, sums, rows, n, sum_blocks, part, dgate, D,
                       chunks);
}

}  // namespace pdt
