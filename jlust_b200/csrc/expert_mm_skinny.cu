// expert_mm_skinny.cu -- the grouped and dense products for a few rows a group
// (decode steps, single tokens): the weights are read once and nothing else
// costs, so the kernel is a stream over W with the rows' values beside it.
//
// A CTA takes a run of up to 8 rows of one group (16 where F32 has more) and one
// tile of columns; the rows sit in shared memory as fp32.  Row-major W: 8 lanes
// read 128 contiguous bytes of one row of W, 32 rows of W a pass; a thread
// keeps the sums of its 16 bytes of columns for all rows, and each weight it
// loads meets every row.  Column-major W: 8 lanes read 128 bytes along K, a
// thread holds 4 columns.  The inner dimension is split over the CTAs of a
// cluster when there are few tiles, and the parts are added through
// distributed shared memory in rank order: one launch, no workspace, the same
// order on every run.  Unaligned W is read one element a lane.
//
// Bound: HBM (L2 for repeated weights).  Sums are fp32 FMAs, one rounding to
// the value type.
#include "expert_mm.cuh"

#include <cooperative_groups.h>

namespace jlb {

JLB_DEFINE_DEV_ERROR(emm_skinny)

namespace emm {

namespace cg = cooperative_groups;

constexpr int kSkThreads = 256, kSkWarps = 8;
constexpr int kSkK = 1024;                 // inner elements of x staged at a time
constexpr int kSkCols = 4;                 // columns a thread holds for column-major W

// Tile width: VEC values a lane (16 bytes, or one), LX lanes side by side.
template <typename T, bool COL, int VEC>
struct SkShape {
    static constexpr int kLX = VEC > 1 ? 8 : COL ? 32 / (int)sizeof(T) : 32;
    static constexpr int kTile = COL ? kSkCols * (32 / kLX) : kLX * VEC;
};

// VEC values as they lie in memory, and their fp32 values.
template <typename T, int VEC>
struct SkRaw {
    uint4 q;
    T one;
};
template <typename T, int VEC>
__device__ __forceinline__ void sk_fetch(SkRaw<T, VEC> &r, const T *p, int n) {
    if constexpr (VEC == 1) {
        r.one = n > 0 ? *p : from_f32<T>(0.0f);
    } else if (n >= VEC) {
        r.q = __ldg(reinterpret_cast<const uint4 *>(p));
    } else {                                       // the matrix's edge: the rest is zero
        T v[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = i < n ? p[i] : from_f32<T>(0.0f);
        r.q = *reinterpret_cast<const uint4 *>(v);
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void sk_value(const SkRaw<T, VEC> &r, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = to_f32(r.one);
    } else {
        const uint32_t w[4] = {r.q.x, r.q.y, r.q.z, r.q.w};
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            v[i] = sizeof(T) == 4 ? __uint_as_float(w[i % 4])
                                  : __uint_as_float(i % 2 ? w[i / 2 % 4] & 0xffff0000u : w[i / 2 % 4] << 16);
    }
}

// Sums of MR rows over inner elements [k0, k1), this thread's part; the CTA's
// sums end in red[0 .. MR * tile).
template <typename T, bool COL, int VEC, int MR>
__device__ __forceinline__ void sk_rows(const Product &P, const T *w, int64_t n0, int row, int nrows, int64_t k0,
                                        int64_t k1, float *xs, float *red, bool &bad) {
    using S = SkShape<T, COL, VEC>;
    constexpr int LX = S::kLX, CT = S::kTile;
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp, lx = lane % LX;
    constexpr int NS = COL ? kSkCols : VEC;        // sums a row and thread
    float acc[MR][NS];
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int c = 0; c < NS; ++c) acc[m][c] = 0.0f;
    // loads a thread has under way (column-major: times four)
    constexpr int U = !COL ? MR <= 8 ? 8 : 4 : VEC == 1 ? 4 : MR <= 4 ? 2 : 1;
    constexpr int kStep = U * (COL ? kSkWarps * LX * VEC : kSkThreads / LX);
    static_assert(kSkK % kStep == 0, "a staged part is a whole number of steps");
    int src[MR];                                   // the rows in x, -1: none
#pragma unroll
    for (int m = 0; m < MR; ++m) {
        src[m] = -1;
        if (m < nrows) {
            int64_t s = row + m;
            if (P.rows) s = (int64_t)__ldg(P.rows + s) - P.base;
            if (s < 0 || s >= P.T) bad = true;
            else src[m] = (int)s;
        }
    }
    for (int64_t kc = k0; kc < k1; kc += kSkK) {
        const int kn = (int)(k1 - kc < kSkK ? k1 - kc : kSkK);
        __syncthreads();                           // the values of the step before are used
        // past kn the rows hold zeros, up to a whole step of the loops below
        const int kp = min(kSkK, (kn + kStep - 1) / kStep * kStep);
        for (int k = threadIdx.x; k < kp; k += kSkThreads) {
            float v[MR];
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                v[m] = 0.0f;
                if (src[m] >= 0 && k < kn) v[m] = to_f32(((const T *)P.x)[(int64_t)src[m] * P.ldx + kc + k]);
            }
            if (!COL && MR % 4 == 0) {
#pragma unroll
                for (int m = 0; m < MR; m += 4)
                    *reinterpret_cast<float4 *>(xs + k * MR + m) = make_float4(v[m], v[m + 1], v[m + 2], v[m + 3]);
            } else {
#pragma unroll
                for (int m = 0; m < MR; ++m) xs[COL ? m * (kSkK + 8) + k : k * MR + m] = v[m];
            }
        }
        __syncthreads();
        // U loads are on their way before the first is used
        if (!COL) {
            constexpr int KY = kSkThreads / LX;    // rows of W a pass
            const int ky = threadIdx.x / LX, n = (int)min((int64_t)VEC, P.N - (n0 + lx * VEC));
            const T *p = w + kc * P.ldw + n0 + lx * VEC;
            for (int kb = ky; kb < kn && n > 0; kb += U * KY) {
                SkRaw<T, VEC> raw[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int k = kb + u * KY;
                    sk_fetch<T, VEC>(raw[u], p + (int64_t)k * P.ldw, k < kn ? n : 0);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int k = kb + u * KY;
                    float v[VEC], xv[MR];
                    sk_value<T, VEC>(raw[u], v);
                    if constexpr (MR % 4 == 0) {
#pragma unroll
                        for (int m = 0; m < MR; m += 4)
                            *reinterpret_cast<float4 *>(xv + m) = *reinterpret_cast<const float4 *>(xs + k * MR + m);
                    } else {
#pragma unroll
                        for (int m = 0; m < MR; ++m) xv[m] = xs[k * MR + m];
                    }
#pragma unroll
                    for (int m = 0; m < MR; ++m)
#pragma unroll
                        for (int c = 0; c < VEC; ++c) acc[m][c] = fmaf(xv[m], v[c], acc[m][c]);
                }
            }
        } else {
            constexpr int KP = LX * VEC;           // inner elements a warp's pass
            const T *p[kSkCols];
#pragma unroll
            for (int c = 0; c < kSkCols; ++c) {
                const int64_t n = n0 + (lane / LX) + c * (32 / LX);
                p[c] = w + (n < P.N ? n : n0) * P.ldw + kc;
            }
            for (int kb = warp * KP + lx * VEC; kb < kn; kb += U * kSkWarps * KP) {
                SkRaw<T, VEC> raw[U][kSkCols];
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int c = 0; c < kSkCols; ++c) {
                        const int k = kb + u * kSkWarps * KP;
                        sk_fetch<T, VEC>(raw[u][c], p[c] + k, kn - k);
                    }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int k = kb + u * kSkWarps * KP;
                    float v[kSkCols][VEC];
#pragma unroll
                    for (int c = 0; c < kSkCols; ++c) sk_value<T, VEC>(raw[u][c], v[c]);
#pragma unroll
                    for (int m = 0; m < MR; ++m) {
                        float xv[VEC];
                        if constexpr (VEC % 4 == 0) {
#pragma unroll
                            for (int i = 0; i < VEC; i += 4)
                                *reinterpret_cast<float4 *>(xv + i) = *reinterpret_cast<const float4 *>(xs + m * (kSkK + 8) + k + i);
                        } else {
#pragma unroll
                            for (int i = 0; i < VEC; ++i) xv[i] = xs[m * (kSkK + 8) + k + i];
                        }
#pragma unroll
                        for (int c = 0; c < kSkCols; ++c)
#pragma unroll
                            for (int i = 0; i < VEC; ++i) acc[m][c] = fmaf(xv[i], v[c][i], acc[m][c]);
                    }
                }
            }
        }
    }
    // the warp's sums, then the warps' in order
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int c = 0; c < NS; ++c) {
            float s = acc[m][c];
            if (COL) {
#pragma unroll
                for (int o = 1; o < LX; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                if (lx == 0) red[(warp * MR + m) * CT + lane / LX + c * (32 / LX)] = s;
            } else {
#pragma unroll
                for (int o = LX; o < kWarp; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                if (lane < LX) red[(warp * MR + m) * CT + lx * VEC + c] = s;
            }
        }
    __syncthreads();
    for (int o = threadIdx.x; o < MR * CT; o += kSkThreads) {
        float s = red[o];
#pragma unroll
        for (int q = 1; q < kSkWarps; ++q) s += red[q * MR * CT + o];
        red[o] = s;
    }
}

// The rows of this CTA: the blockIdx.x-th run of up to MAXR rows, counted over
// the groups in order; false when there are fewer.  A call of 2 rows over 32
// experts launches two runs and not 32 groups (2048 x 4096 bf16: 8.9 against 21
// us), and a group with many rows has them side by side.  One CTA looks at all
// the ranges and reports those that had to be corrected.
template <int MAXR>
__device__ __forceinline__ bool sk_run(const Product &P, int64_t &e, int &row, int &nrows, bool &bad) {
    __shared__ int found, counts[kSkWarps], its_row, its_rows;
    const bool first = blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0;
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    if (threadIdx.x == 0) found = -1;
    int left = blockIdx.x;                            // runs still to pass
    bool done = false;
    for (int64_t e0 = 0; e0 < P.E && (!done || first); e0 += kSkThreads) {
        const int64_t g = e0 + threadIdx.x;
        int lo = 0, hi = 0;
        if (g < P.E) {
            group_rows(P.rowptr, P.base, P.S, g, lo, hi);
            if (first) bad |= group_bad(P.rowptr, P.base, P.S, g);
        }
        const int runs = (hi - lo + MAXR - 1) / MAXR;
        int upto = runs;                              // of this warp's groups, this one's with them
#pragma unroll
        for (int o = 1; o < kWarp; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += u;
        }
        __syncthreads();                              // the counts of the step before are read
        if (lane == kWarp - 1) counts[warp] = upto;
        __syncthreads();
        int before = upto - runs, all = 0;
#pragma unroll
        for (int q = 0; q < kSkWarps; ++q) {
            if (q < warp) before += counts[q];
            all += counts[q];
        }
        if (!done && left >= before && left < before + runs) {
            found = (int)g;
            its_row = lo + (left - before) * MAXR;
            its_rows = min(MAXR, hi - its_row);
        }
        if (left < all) done = true;
        else if (!done) left -= all;
    }
    __syncthreads();
    e = found;
    row = its_row;
    nrows = its_rows;
    return found >= 0;
}

// MAXR: rows taken at a time.
template <typename T, bool COL, int VEC, int MAXR>
__global__ void __launch_bounds__(kSkThreads, MAXR <= 2 ? 4 : 2)
product_skinny(const __grid_constant__ Product P, int splits) {
    using S = SkShape<T, COL, VEC>;
    constexpr int CT = S::kTile;
    extern __shared__ __align__(16) float sk_smem[];
    float *xs = sk_smem;                              // MAXR x (kSkK + 8)
    float *red = sk_smem + MAXR * (kSkK + 8);         // kSkWarps x MAXR x CT
    const int64_t n0 = (int64_t)blockIdx.y * CT;
    bool bad = false;
    int64_t e = 0;
    int row = blockIdx.x * MAXR, nr = (int)min((int64_t)MAXR, P.S - row);
    const bool live = P.rowptr ? sk_run<MAXR>(P, e, row, nr, bad) : true;
    if (P.rowptr && blockIdx.z == 0) {                // rows of no group are zero
        int a, end;
        group_rows(P.rowptr, P.base, P.S, P.E - 1, a, end);
        for (int64_t r = (int64_t)end + blockIdx.x; r < P.S; r += gridDim.x)
            for (int c = threadIdx.x; c < CT && n0 + c < P.N; c += kSkThreads) {
                ((T *)P.y)[r * P.ldy + n0 + c] = from_f32<T>(0.0f);
                if (P.z) ((T *)P.z)[r * P.ldz + n0 + c] = from_f32<T>(0.0f);
            }
    }
    // this CTA's part of the inner dimension, in whole 16-byte groups
    const int64_t share = (ceil_div(P.K, splits) + 63) / 64 * 64;
    const int64_t k0 = min(P.K, share * blockIdx.z), k1 = min(P.K, k0 + share);
    const T *w = (const T *)P.w + e * P.w_stride;
    cg::cluster_group cluster = cg::this_cluster();
    if (live) {                                       // the same for a cluster's CTAs
        if (nr == 1) sk_rows<T, COL, VEC, 1>(P, w, n0, row, nr, k0, k1, xs, red, bad);
        else if (MAXR == 2 || nr == 2) sk_rows<T, COL, VEC, 2>(P, w, n0, row, nr, k0, k1, xs, red, bad);
        else if (nr <= 4) sk_rows<T, COL, VEC, MAXR < 4 ? MAXR : 4>(P, w, n0, row, nr, k0, k1, xs, red, bad);
        else if (MAXR <= 8 || nr <= 8) sk_rows<T, COL, VEC, MAXR < 8 ? MAXR : 8>(P, w, n0, row, nr, k0, k1, xs, red, bad);
        else sk_rows<T, COL, VEC, MAXR>(P, w, n0, row, nr, k0, k1, xs, red, bad);
        if (splits > 1) cluster.sync();
        else __syncthreads();
        if (blockIdx.z == 0)
            for (int o = threadIdx.x; o < nr * CT; o += kSkThreads) {
                const int64_t r = row + o / CT, n = n0 + o % CT;
                if (n >= P.N) continue;
                float v = red[o];
                for (int q = 1; q < splits; ++q) v += *cluster.map_shared_rank(red + o, q);
                if (P.bias) v += to_f32(((const T *)P.bias)[e * P.ldb + n]);
                if (P.z) ((T *)P.z)[r * P.ldz + n] = from_f32<T>(v);
                v = act_value<T>(v, P.act);
                if (P.res) v = add_rn(v, to_f32(((const T *)P.res)[r * P.ldr + n]));
                ((T *)P.y)[r * P.ldy + n] = from_f32<T>(v);
            }
        if (splits > 1) cluster.sync();               // the parts are read before they are overwritten
    }
    if (bad) dev_error(DEV_ERR_BOUNDS);
}

// Few rows, measured here against the tensor path.  BF16: one or two; up to
// eight over experts, where the tensor path starts slowly and joins its parts
// in a second launch (8 rows over 8 experts of 2048 x 1024 9.5 against 14.5 us,
// over 32 of 2048 x 4096 33 against 31, over 69 unaligned ones of 512 x 4093 27
// against 52); more for a small W (16 rows over 64 experts of 512 x 1024 6.7
// against 12.9; 4 dense rows of 2048 x 2048 7.5 against 11, 8 of 2049 x 1023
// 7.8 against 14.5, but 4 of 8192 x 8192 45 against 31).
// F32: the tensor path splits W into planes first, four times W's bytes, and
// this one reads W once for each 16 rows of a group: 4096 x 4096, 16 rows 37
// against 63 us, 17 rows 59 and 32 rows 71 against 64; 7296 x 6784, 17 rows 125
// against 166 and 32 rows 204 against 167; 32 experts of 2048 x 1024, 8 rows
// each 105 and 12 rows each 128 against 230; 8 column-major ones of 1024 x 1001,
// 12 rows each 27 against 40.  How the rows lie is not known here; caches cold,
// over 32 experts of 4096 x 4096, 128 rows of one 240 against 323, over four 252
// against 382, over all 445 against 1,488; over 128 of 512 x 1024, 1024 rows of
// one 96 against 63, over all 115 against 218.
bool skinny_ok(const Product &P) {
    if (P.N > 65535 * 8 || P.K == 0 || P.E == 0) return false;    // a tile is 8 columns or more
    if (P.dtype == JLB_BF16) {
        if (P.S <= 2) return true;
        return P.S <= (P.rowptr ? 16 : 8) && ((P.rowptr && P.S <= 8) || P.K * P.N * P.S <= 1 << 25);
    }
    if (!P.rowptr) return P.S <= 24;
    return P.S <= 16 * P.E && P.S <= 1024;
}

template <typename T, bool COL, int VEC, int MAXR>
static int launch_skinny(cudaStream_t st, const Product &P) {
    using S = SkShape<T, COL, VEC>;
    const int64_t tiles = ceil_div(P.N, S::kTile);
    // runs of rows that the groups can have, at most
    const int64_t most = P.rowptr ? P.E + P.S / MAXR : ceil_div(P.S, MAXR), runs = most < P.S ? most : P.S;
    const int64_t live = tiles * (P.rowptr && P.E < runs ? P.E : runs);
    // Parts of the inner dimension, 1 to 8: the fewest rounds of resident CTAs
    // (4 an SM, 2 with more rows' sums) for a part's length, each part at least
    // 128 long and 3 % of overhead.  A power of two: clusters of 3 or 6 CTAs
    // took twice as long (3 rows over 8 experts of 1024 x 1001 bf16 13.2 us,
    // 4 rows 5.0).  Groups' parts have to be resident at once: among runs that
    // turn out empty, clusters in several rounds took two to three times as long
    // (8 F32 experts of 1024 x 1001, one row each, 24 against 8.6 us); a dense
    // product gains by them (3 F32 rows of 7296 x 6784 column-major 64 against 83).
    const int64_t slots = MAXR <= 2 ? 592 : 296;
    int64_t splits = 1;
    double best = 1e30;
    for (int64_t q = 1; q <= 8 && (q == 1 || q <= P.K / 128); q *= 2) {
        if (P.rowptr && q > 1 && live * q > slots) break;
        const double cost = (double)ceil_div(live * q, slots) / q * (1.0 + 0.03 * q);
        if (cost < best) {
            best = cost;
            splits = q;
        }
    }
    const size_t smem = (size_t)(MAXR * (kSkK + 8) + kSkWarps * MAXR * S::kTile) * 4;
    JLB_CUDA(cudaFuncSetAttribute(product_skinny<T, COL, VEC, MAXR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = (unsigned)splits;
    cfg.gridDim = dim3((unsigned)runs, (unsigned)tiles, (unsigned)splits);
    cfg.blockDim = dim3(kSkThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    JLB_CUDA(cudaLaunchKernelEx(&cfg, product_skinny<T, COL, VEC, MAXR>, P, (int)splits));
    return ok();
}

template <typename T, bool COL, int VEC>
static int skinny_rows(cudaStream_t st, const Product &P) {
    if (P.S <= 2) return launch_skinny<T, COL, VEC, 2>(st, P);
    if constexpr (sizeof(T) == 2) {
        if (P.S <= 4) return launch_skinny<T, COL, VEC, 4>(st, P);
    } else {
        if (P.S > (P.rowptr ? 4 * P.E : 8)) return launch_skinny<T, COL, VEC, 16>(st, P);
    }
    return launch_skinny<T, COL, VEC, 8>(st, P);
}

template <typename T>
static int skinny_of(cudaStream_t st, const Product &P) {
    constexpr int V = 16 / (int)sizeof(T);
    const bool vec = aligned16(P.w) && P.ldw % V == 0 && (P.E == 1 || P.w_stride % V == 0);
    if (P.w_order == JLB_ROW_MAJOR)
        return vec ? skinny_rows<T, false, V>(st, P) : skinny_rows<T, false, 1>(st, P);
    return vec ? skinny_rows<T, true, V>(st, P) : skinny_rows<T, true, 1>(st, P);
}

int skinny_product(cudaStream_t st, const Product &P) {
    return P.dtype == JLB_F32 ? skinny_of<float>(st, P) : skinny_of<__nv_bfloat16>(st, P);
}

}  // namespace emm
}  // namespace jlb
