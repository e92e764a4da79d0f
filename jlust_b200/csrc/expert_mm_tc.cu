// expert_mm_tc.cu -- the grouped products on sm_100a tensor cores (bf16
// operands, fp32 sums): tcgen05 products of CTA pairs, operands staged by TMA.
//
// Orientation.  An output matrix out[j][i] (i contiguous in memory) is
// computed as D (256 lanes i) x (up to 256 columns j): the instruction's M is
// fixed at 256 and its N is a run-time field in steps of 32, so the ragged
// dimension -- a group's rows -- goes on N.  A group of r rows takes
// ceil(r / 256) tiles of equal width rounded up to 32, and a decode step's
// few rows cost an instruction of N = 32 instead of a padded tile.
//   product:  i = output column n, j = row p;  A = W[e]^T (256 columns of W x
//     64 of K), B = 64 of K x the tile's rows of x, sums over K.
//   gradient: i, j = the two widths;  A, B = 64 rows of dz and of x, sums over
//     the group's rows.
// Each CTA of a pair stages its 128 lanes of A and its half of B's columns;
// the tensor cores of both read both halves of B, so a 256 x 256 tile moves
// 32 KB a CTA for 64 of the inner dimension (512 tensor cycles at full rate:
// 64 B a cycle, what the L2 delivers to an SM; one CTA alone would need 96).
//
// Lanes of D are neighbouring i, so the epilogue's plain stores of one column
// are 64 contiguous bytes a warp whatever the leading dimension's alignment.
//
// Ragged sums.  The gradient's last 64-row step of a group must not see the
// next group's rows (they may hold NaN): its rows are fetched by TMA row
// gathers (four rows a copy) whose rows past the group lie past the matrix,
// which TMA fills with zeros.  The same gathers fetch rows through `rows`.
//
// Work split: a persistent grid of CTA pairs; pair c takes tiles c, c + G, ...
// numbered group by group from rowptr on the device (each warp role walks 32
// groups at a time), inside a group in column blocks of 8 tiles for L2 reuse.
// Roles (192 threads): warp 0 copies, warp 1 of the leader issues products,
// warps 2-5 read TMEM and store; two TMEM accumulators, so a tile's epilogue
// overlaps the next tile's products.  Every wait is bounded: on expiry the
// device error word is raised and all roles leave.
#include "expert_mm.cuh"
#include "tcgen05.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

namespace jlb {

JLB_DEFINE_DEV_ERROR(emm_tc)

namespace emm {

using namespace tc;

constexpr int kTcThreads = 192;
constexpr int kMaxStages = 10;
constexpr uint32_t kABytes = 128 * 128;                 // 128 lanes x 64 inner, a CTA's half of A
constexpr uint32_t kBox = 64 * 128;                     // 64 x 64 bf16
constexpr int kJBlock = 8;                              // column tiles that share A's tiles in L2
constexpr long long kTcTimeout = 4000000000ll;          // ~2 s

struct TcArgs {
    int base, act;
    int64_t E, S, I, J, Kc;       // I: lanes' extent; J: columns' extent (gradient); Kc: inner (product)
    int64_t glimit;               // rows the gathered matrix has
    const int32_t *rowptr, *rows;
    int gather;                   // product: 1 = B's rows; gradient: 1 = A's, 2 = B's
    int a_past, b_past;           // gradient: a row index past A's / B's matrix
    const __nv_bfloat16 *bias, *res;
    int64_t ldb, ldr;
    __nv_bfloat16 *z, *out;
    int64_t ldz, ldo, out_stride;
    int stages, bn_max;
};

// A pipeline stage: A's half and, in 32-row boxes, B's.
__host__ __device__ inline uint32_t stage_size(int bn_max) { return kABytes + (uint32_t)((bn_max / 2 + 31) / 32) * 4096u; }

struct TcCtl {
    uint64_t full[kMaxStages], empty[kMaxStages], tfull[2], tempty[2], done;
    uint32_t tmem, fills;
    int abort;
};

__device__ __forceinline__ bool tc_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity)) {
        if (*abort_flag) return false;
        if (clock64() - t0 > kTcTimeout) {
            *abort_flag = 1;
            dev_error(DEV_ERR_TIMEOUT);
            return false;
        }
    }
    return true;
}
// The same for a whole warp: every lane gets one answer, so that no lane waits
// at a warp barrier for one that has left.
__device__ __forceinline__ bool tc_wait_warp(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
    return __all_sync(0xffffffffu, tc_wait(bar, parity, abort_flag));
}
__device__ __forceinline__ void tc_drain(uint32_t bar, uint32_t parity) {
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity))
        if (clock64() - t0 > kTcTimeout) {
            dev_error(DEV_ERR_TIMEOUT);
            return;
        }
}

struct Tile {
    int e, lo, hi;      // group and its rows
    int i0, j0, bn;     // first lane, first column (product: relative to lo), columns of the instruction
};

// Walks the tiles in order, 32 groups at a time; every lane of the warp calls.
template <bool GRAD>
struct Walk {
    int64_t e0, before;
    int total, lo, hi, first, tiles, lane, it;
    __device__ void load(const TcArgs &P) {
        lo = hi = tiles = 0;
        if (e0 + lane < P.E) {
            group_rows(P.rowptr, P.base, P.S, e0 + lane, lo, hi);
            tiles = GRAD ? it * (int)((P.J + 255) / 256) : it * col_tiles(hi - lo, P.bn_max);
        }
        int inc = tiles;
#pragma unroll
        for (int o = 1; o < kWarp; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        first = inc - tiles;
        total = __shfl_sync(0xffffffffu, inc, 31);
    }
    // width of a group's column tiles: equal shares rounded up to 32
    static __device__ __forceinline__ int col_width(int r, int bn_max) {
        const int nt = (r + bn_max - 1) / bn_max;
        return ((r + nt - 1) / nt + 31) & ~31;
    }
    static __device__ __forceinline__ int col_tiles(int r, int bn_max) {
        if (r <= 0) return 0;
        const int w = col_width(r, bn_max);
        return (r + w - 1) / w;
    }
    __device__ void init(const TcArgs &P) {
        lane = threadIdx.x % kWarp;
        it = (int)((P.I + 255) / 256);
        e0 = 0;
        before = 0;
        load(P);
    }
    __device__ bool find(const TcArgs &P, int64_t t, Tile &T) {
        while (t >= before + total) {
            before += total;
            e0 += kWarp;
            if (e0 >= P.E) return false;
            load(P);
        }
        const int want = (int)(t - before);
        const int src = __ffs(__ballot_sync(0xffffffffu, want >= first && want < first + tiles)) - 1;
        T.e = (int)e0 + src;
        T.lo = __shfl_sync(0xffffffffu, lo, src);
        T.hi = __shfl_sync(0xffffffffu, hi, src);
        const int l = want - __shfl_sync(0xffffffffu, first, src);
        const int n = __shfl_sync(0xffffffffu, tiles, src) / it;      // column tiles
        const int jb = l / (kJBlock * it), rem = l - jb * kJBlock * it;
        const int w = min(kJBlock, n - kJBlock * jb);
        const int i = rem / w, j = kJBlock * jb + rem - i * w;
        T.i0 = i * 256;
        if (GRAD) {
            T.j0 = j * 256;
            T.bn = P.J - T.j0 > 128 ? 256 : 128;
        } else {
            const int cw = col_width(T.hi - T.lo, P.bn_max);
            T.j0 = j * cw;
            T.bn = min(cw, (T.hi - T.lo - T.j0 + 31) & ~31);
        }
        return true;
    }
};

// One row index of a gather: its row, or one past the matrix (zeros) when the
// row is outside it.
__device__ __forceinline__ int gather_row(const TcArgs &P, int64_t p, int past, bool &bad) {
    const int64_t r = (int64_t)__ldg(P.rows + p) - P.base;
    if (r >= 0 && r < P.glimit) return (int)r;
    bad = true;
    return past;
}

template <int ACT>
__device__ __forceinline__ void store_column(const TcArgs &P, float v, bool has_z, int64_t row, int64_t i, float r) {
    if (has_z) P.z[row * P.ldz + i] = __float2bfloat16_rn(v);
    v = act_value<__nv_bfloat16>(v, ACT) + r;
    P.out[row * P.ldo + i] = __float2bfloat16_rn(v);
}

// 32 columns of one lane: r[c] is column c0 + c.
template <int ACT>
__device__ __forceinline__ void store_chunk(const TcArgs &P, const uint32_t (&r)[32], float bias, int64_t row0, int n,
                                            int64_t i) {
    float add[32];
#pragma unroll
    for (int c = 0; c < 32; ++c) add[c] = P.res && c < n ? __bfloat162float(P.res[(row0 + c) * P.ldr + i]) : 0.0f;
#pragma unroll
    for (int c = 0; c < 32; ++c)
        if (c < n) store_column<ACT>(P, __uint_as_float(r[c]) + bias, P.z != nullptr, row0 + c, i, add[c]);
}

template <bool A_MN, bool GRAD>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTcThreads, 1)
product_tc(const __grid_constant__ CUtensorMap mA, const __grid_constant__ CUtensorMap mB,
           const __grid_constant__ CUtensorMap mAg, const __grid_constant__ CUtensorMap mBg,
           const __grid_constant__ TcArgs P) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t tiles_u32 = (raw + 1023u) & ~1023u;
    const uint32_t stage_bytes = stage_size(P.bn_max);
    TcCtl *ctl = reinterpret_cast<TcCtl *>(smem_raw + (tiles_u32 - raw) + (size_t)P.stages * stage_bytes);
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    const uint32_t rank = cluster_rank();
    const int64_t pair = blockIdx.x / 2, pairs = gridDim.x / 2;
    volatile int *abort_flag = &ctl->abort;

    if (threadIdx.x == 0) {
        for (int s = 0; s < P.stages; ++s) {
            mbar_init(smem_u32(&ctl->full[s]), 1);
            mbar_init(smem_u32(&ctl->empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&ctl->tfull[b]), 1);
            mbar_init(smem_u32(&ctl->tempty[b]), 8);      // four epilogue warps of each CTA
        }
        mbar_init(smem_u32(&ctl->done), 1);
        ctl->abort = 0;
        ctl->fills = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) alloc_pair(smem_u32(&ctl->tmem), 512);
    fence_before();
    __syncthreads();
    cluster_sync();
    fence_after();
    const uint32_t tmem = ctl->tmem;

    if (warp == 0) {
        // ------------------------------------------------------------ copies
        const uint32_t full0 = map_rank(smem_u32(&ctl->full[0]), 0);
        int stage = 0;
        uint32_t pe = 1u, fills = 0;
        bool ok = true, bad = false;
        if (blockIdx.x == 0)
            for (int64_t e = lane; e < P.E; e += kWarp) bad |= group_bad(P.rowptr, P.base, P.S, e);
        Walk<GRAD> walk;
        walk.init(P);
        Tile T;
        for (int64_t t = pair; ok && walk.find(P, t, T); t += pairs) {
            const int a0 = T.i0 + (int)rank * 128;
            if (!GRAD) {
                const int bh = T.bn / 2, nkb = (int)((P.Kc + 63) / 64);
                const int64_t b0 = (int64_t)T.lo + T.j0 + rank * bh;
                int gi[4];
                if (P.gather)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int64_t p = b0 + lane * 4 + q;
                        gi[q] = lane * 4 + q < bh && p < T.hi ? gather_row(P, p, P.b_past, bad) : P.b_past;
                    }
                const int boxes = (bh + 31) / 32;
                const uint32_t bytes = 2u * (kABytes + (P.gather ? (uint32_t)bh * 128u : (uint32_t)boxes * 4096u));
                for (int kb = 0; kb < nkb; ++kb) {
                    if (!tc_wait_warp(smem_u32(&ctl->empty[stage]), pe, abort_flag)) { ok = false; break; }
                    const uint32_t sA = tiles_u32 + (uint32_t)stage * stage_bytes, sB = sA + kABytes;
                    const uint32_t full = full0 + (uint32_t)stage * 8u;
                    if (lane == 0) {
                        if (rank == 0) mbar_expect_tx(smem_u32(&ctl->full[stage]), bytes);
                        if (A_MN) {
                            tma_3d(sA, &mA, full, a0, kb * 64, T.e);
                            tma_3d(sA + kBox, &mA, full, a0 + 64, kb * 64, T.e);
                        } else {
                            tma_3d(sA, &mA, full, kb * 64, a0, T.e);
                        }
                        if (!P.gather)
                            for (int x = 0; x < boxes; ++x)
                                tma_2d(sB + (uint32_t)x * 4096u, &mB, full, kb * 64, (int)b0 + 32 * x);
                    }
                    __syncwarp();
                    if (P.gather && lane * 4 < bh) tma_gather4(sB + (uint32_t)lane * 512u, &mBg, full, kb * 64, gi);
                    ++fills;
                    if (++stage == P.stages) { stage = 0; pe ^= 1u; }
                }
            } else {
                const int nb = T.bn / 128, rows = T.hi - T.lo, nkb = (rows + 63) / 64;
                const int bj0 = T.j0 + (int)rank * (T.bn / 2);
                const uint32_t bytes = 2u * (kABytes + (uint32_t)nb * kBox);
                // lane l gathers rows 4*(l%16).. of the l/16-th 64-column box
                const int box = lane / 16, r4 = (lane % 16) * 4;
                for (int kb = 0; kb < nkb; ++kb) {
                    const bool tail = rows - kb * 64 < 64;
                    const bool ga = tail || P.gather == 1, gb = tail || P.gather == 2;
                    const int64_t p0 = (int64_t)T.lo + kb * 64;
                    int gia[4], gib[4];
                    if (ga || gb)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int64_t p = p0 + r4 + q;
                            const bool in = p < T.hi;
                            gia[q] = !in ? P.a_past : P.gather == 1 ? gather_row(P, p, P.a_past, bad) : (int)p;
                            gib[q] = !in ? P.b_past : P.gather == 2 ? gather_row(P, p, P.b_past, bad) : (int)p;
                        }
                    if (!tc_wait_warp(smem_u32(&ctl->empty[stage]), pe, abort_flag)) { ok = false; break; }
                    const uint32_t sA = tiles_u32 + (uint32_t)stage * stage_bytes, sB = sA + kABytes;
                    const uint32_t full = full0 + (uint32_t)stage * 8u;
                    if (lane == 0) {
                        if (rank == 0) mbar_expect_tx(smem_u32(&ctl->full[stage]), bytes);
                        if (!ga) {
                            tma_2d(sA, &mA, full, a0, (int)p0);
                            tma_2d(sA + kBox, &mA, full, a0 + 64, (int)p0);
                        }
                        if (!gb)
                            for (int x = 0; x < nb; ++x)
                                tma_2d(sB + (uint32_t)x * kBox, &mB, full, bj0 + 64 * x, (int)p0);
                    }
                    __syncwarp();
                    const uint32_t at = (uint32_t)box * kBox + (uint32_t)(lane % 16) * 512u;
                    if (ga) tma_gather4(sA + at, &mAg, full, a0 + 64 * box, gia);
                    if (gb && box < nb) tma_gather4(sB + at, &mBg, full, bj0 + 64 * box, gib);
                    ++fills;
                    if (++stage == P.stages) { stage = 0; pe ^= 1u; }
                }
            }
        }
        if (bad) dev_error(DEV_ERR_BOUNDS);
        if (lane == 0) ctl->fills = fills;
    } else if (warp == 1) {
        // ------------------------------------------- products (leader's warp)
        if (rank == 0) {
            int stage = 0, buf = 0;
            uint32_t pf = 0, te[2] = {1u, 1u};
            bool ok = true;
            const uint64_t a_desc = operand_desc(tiles_u32, A_MN ? kBox : 16u, 1024u);
            const uint64_t b_desc = operand_desc(tiles_u32 + kABytes, GRAD ? kBox : 16u, 1024u);
            Walk<GRAD> walk;
            walk.init(P);
            Tile T;
            for (int64_t t = pair; ok && walk.find(P, t, T); t += pairs) {
                const int nkb = GRAD ? (T.hi - T.lo + 63) / 64 : (int)((P.Kc + 63) / 64);
                if (nkb == 0) continue;                       // the epilogue writes zeros
                if (!tc_wait_warp(smem_u32(&ctl->tempty[buf]), te[buf], abort_flag)) break;
                te[buf] ^= 1u;
                fence_after();
                const uint32_t idesc = instr_desc(256, (uint32_t)T.bn, A_MN, GRAD);
                for (int kb = 0; kb < nkb; ++kb) {
                    if (!tc_wait_warp(smem_u32(&ctl->full[stage]), pf, abort_flag)) { ok = false; break; }
                    fence_after();
                    if (lane == 0) {
                        const uint64_t off = (uint64_t)(((uint32_t)stage * stage_bytes) >> 4);
                        mma_pair_k64<A_MN ? 128u : 2u, GRAD ? 128u : 2u>(tmem + (uint32_t)buf * 256u, a_desc + off,
                                                                        b_desc + off, idesc, kb > 0);
                        commit_pair(smem_u32(&ctl->empty[stage]));
                        if (kb == nkb - 1) commit_pair(smem_u32(&ctl->tfull[buf]));
                    }
                    __syncwarp();
                    if (++stage == P.stages) { stage = 0; pf ^= 1u; }
                }
                buf ^= 1;
            }
            if (lane == 0) commit_pair(smem_u32(&ctl->done));
            __syncwarp();
        }
    } else {
        // ----------------------------------------------------------- epilogue
        const int qd = warp & 3;
        uint32_t tf[2] = {0u, 0u};
        int buf = 0;
        bool ok = true;
        const uint32_t te0 = map_rank(smem_u32(&ctl->tempty[0]), 0);
        // rows of no group are zero
        if (!GRAD && P.rowptr) {
            int lo, hi;
            group_rows(P.rowptr, P.base, P.S, P.E - 1, lo, hi);
            for (int64_t r = (int64_t)hi + blockIdx.x; r < P.S; r += gridDim.x)
                for (int64_t c = threadIdx.x - 64; c < P.I; c += 128) {
                    P.out[r * P.ldo + c] = __float2bfloat16_rn(0.0f);
                    if (P.z) P.z[r * P.ldz + c] = __float2bfloat16_rn(0.0f);
                }
        }
        Walk<GRAD> walk;
        walk.init(P);
        Tile T;
        for (int64_t t = pair; ok && walk.find(P, t, T); t += pairs) {
            const int64_t i = (int64_t)T.i0 + rank * 128 + qd * 32 + lane;
            const bool in = i < P.I;
            // column 0's row of the output, and its columns
            const int64_t row0 = GRAD ? T.j0 : (int64_t)T.lo + T.j0;
            const int nj = GRAD ? (int)min((int64_t)T.bn, P.J - T.j0) : min(T.bn, T.hi - T.lo - T.j0);
            if (GRAD && T.hi == T.lo) {
                if (in)
                    for (int c = 0; c < nj; ++c)
                        P.out[T.e * P.out_stride + (row0 + c) * P.ldo + i] = __float2bfloat16_rn(0.0f);
                continue;
            }
            const float bias = !GRAD && P.bias && in ? __bfloat162float(P.bias[T.e * P.ldb + i]) : 0.0f;
            if (!tc_wait_warp(smem_u32(&ctl->tfull[buf]), tf[buf], abort_flag)) { ok = false; break; }
            tf[buf] ^= 1u;
            fence_after();
#pragma unroll 1
            for (int c0 = 0; c0 < nj; c0 += 32) {
                uint32_t r[32];
                __syncwarp();
                JLB_TC_LD32(tmem + ((uint32_t)(qd * 32) << 16) + (uint32_t)(buf * 256 + c0), r);
                wait_ld();
                if (!in) continue;
                const int n = nj - c0;
                if (GRAD) {
                    __nv_bfloat16 *o = P.out + T.e * P.out_stride + (row0 + c0) * P.ldo + i;
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (c < n) o[c * P.ldo] = __float2bfloat16_rn(__uint_as_float(r[c]));
                } else {
                    switch (P.act) {
                        case JLB_ACT_RELU: store_chunk<JLB_ACT_RELU>(P, r, bias, row0 + c0, n, i); break;
                        case JLB_ACT_SILU: store_chunk<JLB_ACT_SILU>(P, r, bias, row0 + c0, n, i); break;
                        case JLB_ACT_GELU: store_chunk<JLB_ACT_GELU>(P, r, bias, row0 + c0, n, i); break;
                        default: store_chunk<JLB_ACT_NONE>(P, r, bias, row0 + c0, n, i);
                    }
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(te0 + (uint32_t)buf * 8u);
            buf ^= 1;
        }
    }

    __syncthreads();
    // every copy has landed and every product is done before shared memory and
    // TMEM go (after an abort some may still be on their way)
    if (threadIdx.x == 0) {
        tc_drain(smem_u32(&ctl->done), 0);
        if (rank == 0 && ctl->abort)
            for (uint32_t s = 0; s < (uint32_t)P.stages && s < ctl->fills; ++s)
                tc_drain(smem_u32(&ctl->full[s]), ((ctl->fills - 1 - s) / (uint32_t)P.stages) & 1u);
    }
    __syncthreads();
    cluster_sync();
    if (warp == 1) {
        fence_after();
        dealloc_pair(tmem, 512);
    }
}

// ------------------------------------------------------------------ host
static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

// rows x cols (x experts) of bf16 as {cols, rows[, experts]}, box {64, box_rows}.
static bool make_map(CUtensorMap *m, const void *p, int64_t cols, int64_t rows, int64_t ld, int64_t experts,
                     int64_t stride, int box_rows) {
    auto fn = encode_fn();
    if (!fn) return false;
    const int rank = experts > 0 ? 3 : 2;
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)experts};
    cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, es[3] = {1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void *>(p), dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static bool tma_matrix(const void *p, int64_t ld) { return aligned16(p) && ld % 8 == 0; }

bool tc_product_ok(const Product &P) {
    return P.dtype == JLB_BF16 && P.K > 0 && P.T > 0 && P.E > 0 && tma_matrix(P.x, P.ldx) && tma_matrix(P.w, P.ldw) &&
           (P.E == 1 || P.w_stride % 8 == 0);
}

bool tc_gradient_ok(const Gradient &G) {
    return G.dtype == JLB_BF16 && G.S > 0 && G.T > 0 && tma_matrix(G.x, G.ldx) && tma_matrix(G.dz, G.lddz);
}

static int device_sms() {
    static int sms = [] {
        int dev = 0, n = 0;
        if (cudaGetDevice(&dev) != cudaSuccess ||
            cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
            n = 148;
        return n;
    }();
    return sms;
}

template <bool A_MN, bool GRAD>
static int launch_tc(cudaStream_t st, const CUtensorMap &a, const CUtensorMap &b, const CUtensorMap &ag,
                     const CUtensorMap &bg, TcArgs &P, int64_t tiles) {
    const uint32_t stage = stage_size(P.bn_max);
    const size_t extra = 1024 + sizeof(TcCtl);
    P.stages = (int)((227 * 1024 - extra) / stage);
    if (P.stages > kMaxStages) P.stages = kMaxStages;
    const size_t smem = (size_t)P.stages * stage + extra;
    JLB_CUDA(cudaFuncSetAttribute(product_tc<A_MN, GRAD>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    int64_t pairs = device_sms() / 2;
    if (tiles < pairs) pairs = tiles;
    product_tc<A_MN, GRAD><<<(unsigned)(2 * pairs), kTcThreads, smem, st>>>(a, b, ag, bg, P);
    JLB_LAUNCH_CHECK("product_tc");
    return ok();
}

// Status, or -1 when the driver refuses a tensor map (the caller takes
// another kernel).
int tc_product(cudaStream_t st, const Product &p) {
    CUtensorMap a, b, bg;
    const bool mn = p.w_order == JLB_ROW_MAJOR;
    const int64_t ws = p.E > 1 ? p.w_stride : (mn ? p.K : p.N) * p.ldw;
    if (!(mn ? make_map(&a, p.w, p.N, p.K, p.ldw, p.E, ws, 64) : make_map(&a, p.w, p.K, p.N, p.ldw, p.E, ws, 128)) ||
        !make_map(&b, p.x, p.K, p.T, p.ldx, 0, 0, 32) || (p.rows && !make_map(&bg, p.x, p.K, p.T, p.ldx, 0, 0, 1)))
        return -1;
    if (!p.rows) bg = b;
    TcArgs P{};
    P.base = p.base;
    P.act = p.act;
    P.E = p.E;
    P.S = p.S;
    P.I = p.N;
    P.Kc = p.K;
    P.glimit = p.T;
    P.rowptr = p.rowptr;
    P.rows = p.rows;
    P.gather = p.rows ? 1 : 0;
    P.b_past = (int)p.T;
    P.bias = (const __nv_bfloat16 *)p.bias;
    P.ldb = p.ldb;
    P.res = (const __nv_bfloat16 *)p.res;
    P.ldr = p.ldr;
    P.z = (__nv_bfloat16 *)p.z;
    P.ldz = p.ldz;
    P.out = (__nv_bfloat16 *)p.y;
    P.ldo = p.ldy;
    P.bn_max = p.S >= 256 ? 256 : (int)((p.S + 31) / 32 * 32);
    const int64_t cols = ceil_div(p.S, P.bn_max) + (p.rowptr ? (p.E < p.S ? p.E : p.S) : 0);
    const int64_t tiles = cols * ceil_div(p.N, 256);
    return mn ? launch_tc<true, false>(st, a, b, a, bg, P, tiles) : launch_tc<false, false>(st, a, b, a, bg, P, tiles);
}

int tc_gradient(cudaStream_t st, const Gradient &g) {
    // dw row-major: lanes = columns n (dz), columns = k (x); column-major: exchanged
    const bool row = g.w_order == JLB_ROW_MAJOR;
    CUtensorMap x, xg, d, dg;
    if (!make_map(&x, g.x, g.K, g.T, g.ldx, 0, 0, 64) || !make_map(&xg, g.x, g.K, g.T, g.ldx, 0, 0, 1) ||
        !make_map(&d, g.dz, g.N, g.S, g.lddz, 0, 0, 64) || !make_map(&dg, g.dz, g.N, g.S, g.lddz, 0, 0, 1))
        return -1;
    TcArgs P{};
    P.base = g.base;
    P.E = g.E;
    P.S = g.S;
    P.I = row ? g.N : g.K;
    P.J = row ? g.K : g.N;
    P.glimit = g.T;
    P.rowptr = g.rowptr;
    P.rows = g.rows;
    P.gather = g.rows ? (row ? 2 : 1) : 0;
    P.a_past = (int)(row ? g.S : g.T);
    P.b_past = (int)(row ? g.T : g.S);
    P.out = (__nv_bfloat16 *)g.dw;
    P.ldo = g.lddw;
    P.out_stride = g.dw_stride;
    P.bn_max = P.J > 128 ? 256 : 128;
    const int64_t tiles = g.E * ceil_div(P.I, 256) * ceil_div(P.J, 256);
    return row ? launch_tc<true, true>(st, d, x, dg, xg, P, tiles) : launch_tc<true, true>(st, x, d, xg, dg, P, tiles);
}

}  // namespace emm
}  // namespace jlb
