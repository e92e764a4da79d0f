// expert_mm_tc.cu -- the grouped products on sm_100a tensor cores (bf16
// operands, fp32 sums): tcgen05 products of CTA pairs, operands staged by TMA.
//
// F32 operands come as three bf16 planes, x = h + m + l exactly (8 bits each),
// and six of the nine products of planes are summed: l h, h l, m m, m h, h m,
// h h; what is left out takes up to 2^-21 of a term, 0.7 * 2^-24 on average,
// always toward zero (the planes are truncated so that all have the value's
// sign and a product that overflows stays an infinity).  The tensor cores' fp32 sums
// truncate (measured here: a relative bias of about 4e-6 after 4096 terms, where
// fp32 FMAs have an error of 2e-7), so a chain of them is kept to 64 inner
// elements, small products first: each 64-wide step's sums are read from TMEM
// and added in registers, rounded to nearest.  An infinity or NaN sits in the
// l plane (with h = +-1), which meets the other operand's h plane alone.
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
// Epilogue.  A thread holds one lane (one i) of 32 columns: bias, activation
// and residual work on 32 independent values.  The rounded results turn
// through shared memory as pairs of columns, so that a thread then holds 8
// neighbouring i of two rows and stores 16-byte vectors.
//
// Gathered rows.  A product's rows fetched through `rows` are copied by four
// loader warps: 16-byte cp.async into the swizzled places a TMA box would fill,
// absent rows zero-filled.
// (TMA row gathers, four rows a copy, ran at 88 cycles a copy: 2549 us for the
// 8192 x 4096 x 16384 product against 1007 us without the gather.)
//
// Ragged sums.  The gradient's last 64-row step of a group must not see the
// next group's rows (they may hold NaN): the same warps wait for the step's
// boxes, on a barrier of their own, and write zeros over its foreign rows
// before the step is reported.
//
// Work split: a persistent grid of CTA pairs over the tiles, numbered group by
// group from rowptr on the device, inside a group in blocks of the column tiles
// whose B stays in L2 while A streams past.  Pair c takes tile c and then c + G,
// c + 2G, ... of equal tiles; ragged groups' tiles differ in cost, and there a
// counter in the workspace hands out the next one (over random skewed groups
// the last pair ends 8 % after the mean, in turn 17 %).  One warp of a CTA finds the tiles, 32
// groups at a time, up to four ahead, and passes them to the other roles
// through a ring in shared memory: found by each role at its tile's start, the
// tensor cores stood still for some 1500 cycles a tile.
// The tiles that do not fill a last round of the G pairs (all of them, when
// there are few) are split along the inner dimension among the pairs; their
// fp32 parts go to the workspace and finish_tc adds them in order and applies
// the epilogue.
// Roles: warp 0 copies, warp 1 of the leader issues products, warps 2-9 read
// TMEM and store, warp 10 finds the tiles, warps 11-14 (only in launches that
// need them) load rows and warp 15 reports their stages to the leader; two TMEM accumulators, so a tile's epilogue
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

constexpr int kEpiWarps = 8;                            // two for each quarter of TMEM's lanes
constexpr int kFindWarp = 2 + kEpiWarps;                // finds the tiles
constexpr int kTcThreads = 32 + kFindWarp * 32;         // without the loaders
constexpr int kLoadWarp = kFindWarp + 1, kLoaders = 128;  // the loader warps
constexpr int kTileRing = 4;                            // tiles found ahead
constexpr int kTickets = 4;                             // numbers on their way to the pair's other CTA
constexpr int kForward = 32;                            // the warp that reports the loaders' stages
constexpr int kPitch = 36;                              // words a pair of columns takes in the epilogue's turn
constexpr uint32_t kTurnBytes = kEpiWarps * 16 * kPitch * 4;
constexpr int kMaxStages = 10;
constexpr uint32_t kABytes = 128 * 128;                 // 128 lanes x 64 inner, a CTA's half of A
constexpr uint32_t kBox = 64 * 128;                     // 64 x 64 bf16
constexpr int64_t kL2Block = 24 << 20;                  // bytes of B that a block of column tiles keeps in L2
constexpr long long kTcTimeout = 4000000000ll;          // ~2 s

struct TcArgs {
    int base, act;
    int64_t E, S, I, J, Kc;       // I: lanes' extent; J: columns' extent (gradient); Kc: inner (product)
    int64_t glimit;               // rows the gathered matrix has
    const int32_t *rowptr, *rows;
    int gather;                   // product: B's rows come through rows
    int vec;                      // out, z and res allow 16-byte vectors
    const __nv_bfloat16 *gb;      // the rows' matrix, for the loader warps
    int pa, pb;                   // F32: coordinate from an operand's plane to the next (A of a product: experts)
    int64_t ldb_;
    const void *bias, *res;       // of the value type
    int64_t ldb, ldr;
    void *z, *out;
    int64_t ldz, ldo, out_stride;
    int stages, bn_max, jblock;
    int a_pair, b_pair;           // mA / mBig: both 64-wide boxes of an operand in one copy
    int pairs, max_splits;        // CTA pairs launched; parts a tile may be split into (> 1: rowptr decides)
    int full, splits;             // tiles not split and the parts of the others, when the host knows
    float *part;                  // one 256 x bn_max fp32 tile for each part
    int *counter;                 // tiles handed out beyond each pair's first; null: in turn
};

// A pipeline stage: A's half and, in 32-row boxes, B's.
__host__ __device__ inline uint32_t stage_size(int bn_max) { return kABytes + (uint32_t)((bn_max / 2 + 31) / 32) * 4096u; }

struct Tile {
    int e, lo, hi;      // group and its rows
    int i0, j0, bn;     // first lane, first column (product: relative to lo), columns of the instruction
    int kb0, kb1;       // 64-wide steps of the inner dimension
    int part;           // where a split tile's sums go, or -1
};

struct TcCtl {
    uint64_t full[kMaxStages], empty[kMaxStages], rows[kMaxStages], go[kMaxStages];
    uint64_t tfull[2], tempty[2], done;
    uint64_t sfull[kTileRing], sempty[kTileRing], tbar[kTickets], tack[kTickets];
    int ticket[kTickets];
    Tile ring[kTileRing];
    uint32_t tmem, fills;
    uint32_t tails, tail_phase;                   // stages a last step used, and their go barriers' phases, a bit each
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

// width of a group's column tiles: equal shares rounded up to 32
__host__ __device__ __forceinline__ int col_width(int r, int bn_max) {
    const unsigned nt = (unsigned)(r + bn_max - 1) / (unsigned)bn_max;
    return (int)((((unsigned)r + nt - 1u) / nt + 31u) & ~31u);
}
__host__ __device__ __forceinline__ int col_tiles(int r, int bn_max) {
    if (r <= bn_max) return r > 0;
    const int w = col_width(r, bn_max);
    return (int)((unsigned)(r + w - 1) / (unsigned)w);
}

// Tiles of the full rounds, and into how many parts each of the rest is split.
__host__ __device__ inline void split_schedule(int all, int pairs, int max_splits, int &full, int &splits) {
    full = (int)((unsigned)all / (unsigned)pairs) * pairs;
    const int rest = all - full;
    splits = rest && max_splits > 1 ? (int)((unsigned)pairs / (unsigned)rest) : 1;
    if (splits > max_splits) splits = max_splits;
    if (splits <= 1) {
        splits = 1;
        full = all;
    }
}

// Walks the tiles in order, 32 groups at a time; every lane of the warp calls.
// 32-bit arithmetic throughout: a launch of few tiles pays for its first
// instructions (with 64-bit divisions 10,000 cycles went by before the first
// copy, now 4,000; as calls of one function 8,000).
template <bool GRAD>
struct Walk {
    int e0, before, total, lo, hi, first, tiles, it, jt;
    int full, splits;                 // tiles not split; parts of each other one

    __device__ __forceinline__ int count(const TcArgs &P, int e, int &a, int &b) const {
        group_rows(P.rowptr, P.base, P.S, e, a, b);
        return GRAD ? it * jt : it * col_tiles(b - a, P.bn_max);
    }
    __device__ __forceinline__ void load(const TcArgs &P) {
        const int lane = threadIdx.x % kWarp;
        lo = hi = tiles = 0;
        if (e0 + lane < (int)P.E) tiles = count(P, e0 + lane, lo, hi);
        int inc = tiles;
        if (P.E > 1)
#pragma unroll
            for (int o = 1; o < kWarp; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += u;
            }
        first = inc - tiles;
        total = __shfl_sync(0xffffffffu, inc, P.E > 1 ? 31 : 0);
    }
    __device__ __forceinline__ void init(const TcArgs &P) {
        it = (int)((P.I + 255) >> 8);
        jt = GRAD ? (int)((unsigned)(P.J + P.bn_max - 1) / (unsigned)P.bn_max) : 1;
        full = P.full;
        splits = P.splits;
        if (P.max_splits > 1) {       // a product whose tiles only rowptr tells
            const int lane = threadIdx.x % kWarp;
            int all = 0;
            for (int e = lane; e < (int)P.E; e += kWarp) {
                int a, b;
                all += count(P, e, a, b);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
            split_schedule(all, P.pairs, P.max_splits, full, splits);
        }
        e0 = 0;
        before = 0;
        load(P);
    }
    __device__ __forceinline__ int steps(const TcArgs &P, const Tile &T) const {
        return GRAD ? (T.hi - T.lo + 63) >> 6 : (int)((P.Kc + 63) >> 6);
    }
    // Work item u of a pair: a whole tile, or a part of one of the rest.
    __device__ __forceinline__ bool find(const TcArgs &P, int u, Tile &T) {
        if (u < full || splits == 1) {
            if (!tile(P, u, T)) return false;
            T.kb0 = 0;
            T.kb1 = steps(P, T);
            T.part = -1;
            return true;
        }
        const unsigned q = (unsigned)(u - full), t = q / (unsigned)splits, sp = q - t * splits;
        if (!tile(P, full + (int)t, T)) return false;
        const unsigned nkb = (unsigned)steps(P, T);    // < 2^25 steps, < 2^7 parts
        T.kb0 = (int)(nkb * sp / splits);
        T.kb1 = (int)(nkb * (sp + 1) / splits);
        T.part = (int)q;
        return true;
    }
    __device__ __forceinline__ bool tile(const TcArgs &P, int t, Tile &T) {
        while (t >= before + total) {
            before += total;
            e0 += kWarp;
            if (e0 >= (int)P.E) return false;
            load(P);
        }
        const int want = t - before;
        int src = 0;
        if (P.E > 1) src = __ffs(__ballot_sync(0xffffffffu, want >= first && want < first + tiles)) - 1;
        T.e = e0 + src;
        T.lo = __shfl_sync(0xffffffffu, lo, src);
        T.hi = __shfl_sync(0xffffffffu, hi, src);
        const int l = want - __shfl_sync(0xffffffffu, first, src);
        // column tiles j, in blocks of jblock, lane tiles i inside a block
        const int cw = GRAD ? P.bn_max : col_width(T.hi - T.lo, P.bn_max);
        const int n = GRAD ? jt : (int)((unsigned)(T.hi - T.lo + cw - 1) / (unsigned)cw);
        int i = l, j = 0;
        if (n > 1) {
            const int jb = n <= P.jblock ? 0 : (int)((unsigned)l / (unsigned)(P.jblock * it));
            const int rem = l - jb * P.jblock * it, w = min(P.jblock, n - P.jblock * jb);
            i = (int)((unsigned)rem / (unsigned)w);
            j = P.jblock * jb + rem - i * w;
        }
        T.i0 = i * 256;
        T.j0 = j * cw;
        if (GRAD) T.bn = P.bn_max > 128 && P.J - T.j0 > 128 ? 256 : 128;
        else T.bn = min(cw, (T.hi - T.lo - T.j0 + 31) & ~31);
        return true;
    }
};

// A role's view of the ring of tiles its CTA's finding warp fills; a tile of
// no columns ends it.
struct TileReader {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ bool next(TcCtl *ctl, Tile &T, volatile int *abort_flag) {
        if (!tc_wait_warp(smem_u32(&ctl->sfull[slot]), phase, abort_flag)) return false;
        T = ctl->ring[slot];
        __syncwarp();
        if (threadIdx.x % kWarp == 0) mbar_arrive_count(smem_u32(&ctl->sempty[slot]), 1);
        if (++slot == kTileRing) { slot = 0; phase ^= 1u; }
        return T.bn != 0;
    }
};

// cp.async of up to 16 bytes; the rest of the 16 is zeroed (bytes == 0: all).
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ void zero16(uint32_t dst) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0) : "memory");
}

// Bytes of the 16 at element `at` of a row of `cols` elements.
__device__ __forceinline__ uint32_t bytes_at(int64_t at, int64_t cols) {
    const int64_t left = cols - at;
    return left >= 8 ? 16u : left > 0 ? (uint32_t)left * 2u : 0u;
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Stores 32 columns of the warp's 32 lanes: v[c] = out[row0 + c][ib + lane],
// columns c < n.
__device__ __forceinline__ void store32(const float (&v)[32], uint32_t *turn, bool vec, __nv_bfloat16 *out,
                                        int64_t ld, int64_t row0, int n, int64_t ib, int64_t I) {
    const int lane = threadIdx.x % kWarp;
    if (!vec) {                                   // 32 neighbouring values a store, no alignment needed
        if (ib + lane < I) {
            __nv_bfloat16 *o = out + row0 * ld + ib + lane;
#pragma unroll
            for (int c = 0; c < 32; ++c)
                if (c < n) o[c * ld] = __float2bfloat16_rn(v[c]);
        }
        return;
    }
#pragma unroll
    for (int c = 0; c < 16; ++c) turn[c * kPitch + lane] = pack2(v[2 * c], v[2 * c + 1]);
    __syncwarp();
    const int pr = lane / 4, oct = (lane % 4) * 8;
    __nv_bfloat16 *o = out + (row0 + 2 * pr) * ld + ib + oct;
    const uint32_t *w = turn + pr * kPitch + oct;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t a[8], lo[4], hi[4];
        *reinterpret_cast<uint4 *>(a) = *reinterpret_cast<const uint4 *>(w + h * 8 * kPitch);
        *reinterpret_cast<uint4 *>(a + 4) = *reinterpret_cast<const uint4 *>(w + h * 8 * kPitch + 4);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            lo[c] = __byte_perm(a[2 * c], a[2 * c + 1], 0x5410);
            hi[c] = __byte_perm(a[2 * c], a[2 * c + 1], 0x7632);
        }
        const int c = 16 * h + 2 * pr;
        if (c < n) *reinterpret_cast<uint4 *>(o + 16 * h * ld) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        if (c + 1 < n) *reinterpret_cast<uint4 *>(o + (16 * h + 1) * ld) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    }
    __syncwarp();
}

// The 32 columns of F32 results, v[c] = out[row0 + c][i] of every lane: 128
// contiguous bytes a store.
__device__ __forceinline__ void store32_f32(const float (&v)[32], float *out, int64_t ld, int64_t row0, int n,
                                            int64_t i, int64_t I) {
    if (i >= I) return;
    float *o = out + row0 * ld + i;
#pragma unroll
    for (int c = 0; c < 32; ++c)
        if (c < n) o[c * ld] = v[c];
}

template <int ACT>
__device__ __forceinline__ void act32_f32(float (&v)[32]) {
#pragma unroll
    for (int c = 0; c < 32; ++c) v[c] = act_value<float>(v[c], ACT);
}

// The epilogue of 32 columns of F32 sums.
template <bool GRAD>
__device__ __forceinline__ void finish32_f32(const TcArgs &P, float (&v)[32], int64_t row0, int n, int64_t i,
                                             float bias, float *out) {
    if (!GRAD) {
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] += bias;
        if (P.z) store32_f32(v, (float *)P.z, P.ldz, row0, n, i, P.I);
        // unrolled: an index that the compiler does not know would put the sums
        // in local memory for the whole kernel
        switch (P.act) {
            case JLB_ACT_RELU: act32_f32<JLB_ACT_RELU>(v); break;
            case JLB_ACT_SILU: act32_f32<JLB_ACT_SILU>(v); break;
            case JLB_ACT_GELU: act32_f32<JLB_ACT_GELU>(v); break;
            default: break;
        }
        if (P.res && i < P.I) {
            const float *q = (const float *)P.res + row0 * P.ldr + i;
#pragma unroll
            for (int c = 0; c < 32; ++c)
                if (c < n) v[c] = add_rn(v[c], q[c * P.ldr]);
        }
    }
    store32_f32(v, out, P.ldo, row0, n, i, P.I);
}

// Every second 32-column chunk of the tile's columns [0, nj), from chunk
// `first` on, of this warp's 32 lanes; column c is output row row0 + c.
template <int ACT, bool GRAD>
__device__ __forceinline__ void store_tile(const TcArgs &P, uint32_t taddr, uint32_t *turn, int first, int64_t row0,
                                           int nj, int64_t ib, float bias, __nv_bfloat16 *out) {
    const int64_t i = ib + threadIdx.x % kWarp;
    const bool vec = P.vec && ib + 32 <= P.I;
#pragma unroll 1
    for (int c0 = first * 32; c0 < nj; c0 += 64) {
        const int n = nj - c0;
        uint32_t r[32];
        __syncwarp();
        JLB_TC_LD32(taddr + (uint32_t)c0, r);
        wait_ld();
        float v[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = __uint_as_float(r[c]) + (GRAD ? 0.0f : bias);
        if (!GRAD) {
            if (P.z) store32(v, turn, vec, (__nv_bfloat16 *)P.z, P.ldz, row0 + c0, n, ib, P.I);
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = act_value<__nv_bfloat16>(v[c], ACT);
            if (P.res && i < P.I) {
                const __nv_bfloat16 *q = (const __nv_bfloat16 *)P.res + (row0 + c0) * P.ldr + i;
#pragma unroll
                for (int c = 0; c < 32; ++c)
                    if (c < n) v[c] = add_rn(v[c], __bfloat162float(q[c * P.ldr]));
            }
        }
        store32(v, turn, vec, out, P.ldo, row0 + c0, n, ib, P.I);
    }
    __syncwarp();
}

template <bool A_MN, bool GRAD, typename T_>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTcThreads + kLoaders + kForward, 1)
product_tc(const __grid_constant__ CUtensorMap mA, const __grid_constant__ CUtensorMap mB,
           const __grid_constant__ CUtensorMap mBig, const __grid_constant__ CUtensorMap mMid,
           const __grid_constant__ TcArgs P) {
    constexpr bool F32 = sizeof(T_) == 4;
    constexpr int kPlanes = F32 ? 3 : 1;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t tiles_u32 = (raw + 1023u) & ~1023u;
    const uint32_t stage_bytes = stage_size(P.bn_max);
    uint8_t *after = smem_raw + (tiles_u32 - raw) + (size_t)P.stages * stage_bytes;
    uint32_t *turns = reinterpret_cast<uint32_t *>(after);
    TcCtl *ctl = reinterpret_cast<TcCtl *>(after + kTurnBytes);
    const bool loaders = blockDim.x > kTcThreads;
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;
    volatile int *abort_flag = &ctl->abort;

    if (threadIdx.x == 0) {
        for (int s = 0; s < P.stages; ++s) {
            mbar_init(smem_u32(&ctl->full[s]), loaders ? 3 : 1);   // the leader's copies; both CTAs' rows
            mbar_init(smem_u32(&ctl->rows[s]), kLoaders);
            mbar_init(smem_u32(&ctl->go[s]), 1);
            mbar_init(smem_u32(&ctl->empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&ctl->tfull[b]), 1);
            mbar_init(smem_u32(&ctl->tempty[b]), 2 * kEpiWarps);
        }
        mbar_init(smem_u32(&ctl->done), 1);
        for (int b = 0; b < kTickets; ++b) {
            mbar_init(smem_u32(&ctl->tbar[b]), 1);
            mbar_init(smem_u32(&ctl->tack[b]), 1);
        }
        for (int b = 0; b < kTileRing; ++b) {
            mbar_init(smem_u32(&ctl->sfull[b]), 1);
            // the warps that read it: copies, epilogue, the leader's products, loaders and their report
            mbar_init(smem_u32(&ctl->sempty[b]), 1 + kEpiWarps + (rank == 0 ? 1 : 0) + (loaders ? (kLoaders + kForward) / kWarp : 0));
        }
        ctl->abort = 0;
        ctl->fills = 0;
        ctl->tails = ctl->tail_phase = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) alloc_pair(smem_u32(&ctl->tmem), 512);
    fence_before();
    __syncthreads();
    cluster_sync_relaxed();               // the barriers' set-up is fenced above
    fence_after();
    const uint32_t tmem = ctl->tmem;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp == 0) {
        // ------------------------------------------------------------ copies
        const uint32_t full0 = map_rank(smem_u32(&ctl->full[0]), 0);
        int stage = 0;
        uint32_t pe = 1u, fills = 0, tails = 0, tail_phase = 0;
        bool ok = true, bad = false;
        if (blockIdx.x == 0)
            for (int64_t e = lane; e < P.E; e += kWarp) bad |= group_bad(P.rowptr, P.base, P.S, e);
        TileReader tiles;
        Tile T;
        while (ok && tiles.next(ctl, T, abort_flag)) {
            const int a0 = T.i0 + (int)rank * 128;
            const int bh = T.bn / 2, boxes = (bh + 31) / 32;           // product: B's rows, in 32-row boxes
            const int64_t b0 = (int64_t)T.lo + T.j0 + rank * bh;
            const int nb = T.bn / 128, bj0 = T.j0 + (int)rank * bh;    // gradient: B's 64-column boxes
            for (int k = T.kb0 * kPlanes; k < T.kb1 * kPlanes; ++k) {
                const int kb = k / kPlanes, plane = k - kb * kPlanes;
                if (!tc_wait_warp(smem_u32(&ctl->empty[stage]), pe, abort_flag)) { ok = false; break; }
                const uint32_t sA = tiles_u32 + (uint32_t)stage * stage_bytes, sB = sA + kABytes;
                const uint32_t full = full0 + (uint32_t)stage * 8u;
                if (!GRAD) {
                    const int e = T.e + plane * P.pa, r0 = (int)b0 + plane * P.pb;
                    if (rank == 0)
                        mbar_expect_tx(smem_u32(&ctl->full[stage]),
                                       2u * (kABytes + (P.gather ? 0u : (uint32_t)boxes * 4096u)));
                    if (!A_MN) {
                        tma_3d(sA, &mA, full, kb * 64, a0, e);
                    } else if (P.a_pair) {
                        tma_4d(sA, &mA, full, 0, kb * 64, a0 / 64, e);
                    } else {
                        tma_3d(sA, &mA, full, a0, kb * 64, e);
                        tma_3d(sA + kBox, &mA, full, a0 + 64, kb * 64, e);
                    }
                    if (!P.gather) {                       // few copies: each costs the issuing thread
                        if (boxes == 4) tma_2d(sB, &mBig, full, kb * 64, r0);
                        else if (boxes >= 2) tma_2d(sB, &mMid, full, kb * 64, r0);
                        if (boxes & 1) tma_2d(sB + (uint32_t)(boxes - 1) * 4096u, &mB, full, kb * 64, r0 + 32 * (boxes - 1));
                    }
                } else {
                    // a group's last step goes through the loader warps' hands
                    const bool tail = T.hi - T.lo - kb * 64 < 64;
                    const uint32_t to = tail ? smem_u32(&ctl->go[stage]) : full;
                    const uint32_t bytes = kABytes + (uint32_t)nb * kBox;
                    const int pa = T.lo + kb * 64 + plane * P.pa, pb = T.lo + kb * 64 + plane * P.pb;
                    if (rank == 0) mbar_expect_tx(smem_u32(&ctl->full[stage]), tail ? 0u : 2u * bytes);
                    if (rank == 0 && !tail)                // no hands: their arrivals
                        mbar_arrive_elect(smem_u32(&ctl->full[stage]), 2);
                    if (tail) {
                        mbar_expect_tx(to, bytes);
                        tails |= 1u << stage;
                        tail_phase ^= 1u << stage;
                    }
                    if (P.a_pair) {
                        tma_3d(sA, &mA, to, 0, pa, a0 / 64);
                    } else {
                        tma_2d(sA, &mA, to, a0, pa);
                        tma_2d(sA + kBox, &mA, to, a0 + 64, pa);
                    }
                    if (nb == 2 && P.b_pair) {
                        tma_3d(sB, &mBig, to, 0, pb, bj0 / 64);
                    } else {
                        for (int x = 0; x < nb; ++x)
                            tma_2d(sB + (uint32_t)x * kBox, &mB, to, bj0 + 64 * x, pb);
                    }
                }
                ++fills;
                if (++stage == P.stages) { stage = 0; pe ^= 1u; }
            }
        }
        // every stage's last release has arrived: none can reach this CTA later
        if (lane == 0)
            for (uint32_t n = 0; ok && n < (uint32_t)P.stages && n < fills; ++n) {
                if (fills < (uint32_t)P.stages) {
                    ok = tc_wait(smem_u32(&ctl->empty[n]), 0u, abort_flag);
                } else {
                    ok = tc_wait(smem_u32(&ctl->empty[stage]), pe, abort_flag);
                    if (++stage == P.stages) { stage = 0; pe ^= 1u; }
                }
            }
        __syncwarp();
        if (bad) dev_error(DEV_ERR_BOUNDS);
        if (lane == 0) {
            ctl->fills = fills;
            ctl->tails = tails;
            ctl->tail_phase = tail_phase;
        }
    } else if (warp == 1) {
        // ------------------------------------------- products (leader's warp)
        if (rank == 0) {
            int stage = 0, buf = 0;
            uint32_t pf = 0, te[2] = {1u, 1u};
            bool ok = true;
            const uint64_t a_desc = operand_desc(tiles_u32, A_MN ? kBox : 16u, 1024u);
            const uint64_t b_desc = operand_desc(tiles_u32 + kABytes, GRAD ? kBox : 16u, 1024u);
            TileReader tiles;
            Tile T;
            while (ok && tiles.next(ctl, T, abort_flag)) {
                if (T.kb0 == T.kb1) continue;                 // the epilogue writes zeros
                const uint32_t idesc = instr_desc(256, (uint32_t)T.bn, A_MN, GRAD);
                auto mma = [&](uint32_t a_off, uint32_t b_off, uint32_t first) {
                    mma_pair_k64<A_MN ? 128 : 2, GRAD ? 128 : 2>(tmem + (uint32_t)buf * 256u, (uint32_t)a_desc + a_off,
                                                                 (uint32_t)(a_desc >> 32), (uint32_t)b_desc + b_off,
                                                                 (uint32_t)(b_desc >> 32), idesc, first);
                };
                if (!F32) {
                    if (!tc_wait_warp(smem_u32(&ctl->tempty[buf]), te[buf], abort_flag)) break;
                    te[buf] ^= 1u;
                    fence_after();
                    // the whole warp goes through the loop: converged, its
                    // operands stay in uniform registers
                    for (int kb = T.kb0; kb < T.kb1; ++kb) {
                        if (!tc_wait_warp(smem_u32(&ctl->full[stage]), pf, abort_flag)) { ok = false; break; }
                        fence_after();
                        const uint32_t off = ((uint32_t)stage * stage_bytes) >> 4;
                        mma(off, off, (uint32_t)(kb - T.kb0));
                        commit_pair(smem_u32(&ctl->empty[stage]));
                        if (++stage == P.stages) { stage = 0; pf ^= 1u; }
                    }
                    if (ok) commit_pair(smem_u32(&ctl->tfull[buf]));
                    buf ^= 1;
                } else {
                    // a 64-wide step: its three planes' stages, then six products into a fresh accumulator
                    for (int kb = T.kb0; ok && kb < T.kb1; ++kb) {
                        ok = tc_wait_warp(smem_u32(&ctl->tempty[buf]), te[buf], abort_flag);
                        te[buf] ^= 1u;
                        uint32_t off[3], bar[3];
#pragma unroll
                        for (int q = 0; q < 3; ++q) {
                            ok = ok && tc_wait_warp(smem_u32(&ctl->full[stage]), pf, abort_flag);
                            off[q] = ((uint32_t)stage * stage_bytes) >> 4;
                            bar[q] = smem_u32(&ctl->empty[stage]);
                            if (++stage == P.stages) { stage = 0; pf ^= 1u; }
                        }
                        if (!ok) break;
                        fence_after();
                        mma(off[2], off[0], 0u);
                        mma(off[0], off[2], 1u);
                        mma(off[1], off[1], 1u);
                        mma(off[1], off[0], 1u);
                        mma(off[0], off[1], 1u);
                        mma(off[0], off[0], 1u);
#pragma unroll
                        for (int q = 0; q < 3; ++q) commit_pair(bar[q]);
                        commit_pair(smem_u32(&ctl->tfull[buf]));
                        buf ^= 1;
                    }
                }
            }
            // both accumulators' last releases have arrived: the other CTA's
            // epilogue sends none to a CTA that is gone
#pragma unroll
            for (int b = 0; b < 2; ++b)
                ok = ok && tc_wait_warp(smem_u32(&ctl->tempty[b]), te[b], abort_flag);
            __syncwarp();
            commit_pair(smem_u32(&ctl->done));
        }
    } else if (warp < kFindWarp) {
        // ----------------------------------------------------------- epilogue
        const int qd = warp & 3;
        const int first = (warp - 2) / 4;                 // the 32-column chunks of this parity
        uint32_t *turn = turns + (warp - 2) * 16 * kPitch;
        uint32_t tf[2] = {0u, 0u};
        int buf = 0;
        const uint32_t te0 = map_rank(smem_u32(&ctl->tempty[0]), 0);
        // rows of no group are zero
        if (!GRAD && P.rowptr) {
            int lo, hi;
            group_rows(P.rowptr, P.base, P.S, P.E - 1, lo, hi);
            for (int64_t r = (int64_t)hi + blockIdx.x; r < P.S; r += gridDim.x)
                for (int64_t c = threadIdx.x - 64; c < P.I; c += kEpiWarps * 32) {
                    ((T_ *)P.out)[r * P.ldo + c] = from_f32<T_>(0.0f);
                    if (P.z) ((T_ *)P.z)[r * P.ldz + c] = from_f32<T_>(0.0f);
                }
        }
        TileReader tiles;
        Tile T;
        while (tiles.next(ctl, T, abort_flag)) {
            const int64_t ib = (int64_t)T.i0 + rank * 128 + qd * 32;
            // column 0's row of the output, and its columns
            const int64_t row0 = GRAD ? T.j0 : (int64_t)T.lo + T.j0;
            const int nj = GRAD ? (int)min((int64_t)T.bn, P.J - T.j0) : min(T.bn, T.hi - T.lo - T.j0);
            T_ *out = (T_ *)P.out + (GRAD ? T.e * P.out_stride : 0);
            float *part = T.part >= 0 ? P.part + (int64_t)T.part * 256 * P.bn_max + (ib - T.i0) + lane : nullptr;
            if (T.kb0 == T.kb1) {
                for (int c = first; c < nj; c += 2) {
                    if (part) part[c * 256] = 0.0f;
                    else if (ib + lane < P.I) out[(row0 + c) * P.ldo + ib + lane] = from_f32<T_>(0.0f);
                }
                continue;
            }
            const float bias = !GRAD && P.bias && ib + lane < P.I ? to_f32(((const T_ *)P.bias)[T.e * P.ldb + ib + lane]) : 0.0f;
            if constexpr (F32) {
                // this warp's columns 32 first .. and 64 + 32 first .., step after step
                float acc[2][32];
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int c = 0; c < 32; ++c) acc[q][c] = 0.0f;
                bool ok = true;
                for (int kb = T.kb0; kb < T.kb1; ++kb) {
                    ok = tc_wait_warp(smem_u32(&ctl->tfull[buf]), tf[buf], abort_flag);
                    if (!ok) break;
                    tf[buf] ^= 1u;
                    fence_after();
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int c0 = first * 32 + q * 64;
                        if (c0 >= nj) continue;
                        uint32_t r[32];
                        __syncwarp();
                        JLB_TC_LD32(tmem + ((uint32_t)(qd * 32) << 16) + (uint32_t)(buf * 256 + c0), r);
                        wait_ld();
#pragma unroll
                        for (int c = 0; c < 32; ++c) acc[q][c] += __uint_as_float(r[c]);
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(te0 + (uint32_t)buf * 8u);
                    buf ^= 1;
                }
                if (!ok) break;
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int c0 = first * 32 + q * 64;
                    if (c0 >= nj) continue;
                    if (part) {
#pragma unroll
                        for (int c = 0; c < 32; ++c) part[(c0 + c) * 256] = acc[q][c];
                    } else {
                        finish32_f32<GRAD>(P, acc[q], row0 + c0, nj - c0, ib + lane, bias, (float *)out);
                    }
                }
                continue;
            }
            if (!tc_wait_warp(smem_u32(&ctl->tfull[buf]), tf[buf], abort_flag)) break;
            tf[buf] ^= 1u;
            fence_after();
            const uint32_t taddr = tmem + ((uint32_t)(qd * 32) << 16) + (uint32_t)(buf * 256);
            if (part) {
                for (int c0 = first * 32; c0 < nj; c0 += 64) {
                    uint32_t r[32];
                    __syncwarp();
                    JLB_TC_LD32(taddr + (uint32_t)c0, r);
                    wait_ld();
#pragma unroll
                    for (int c = 0; c < 32; ++c) part[(c0 + c) * 256] = __uint_as_float(r[c]);
                }
            } else if (ib < P.I) {
                switch (GRAD ? JLB_ACT_NONE : P.act) {
                    case JLB_ACT_RELU: store_tile<JLB_ACT_RELU, GRAD>(P, taddr, turn, first, row0, nj, ib, bias, (__nv_bfloat16 *)out); break;
                    case JLB_ACT_SILU: store_tile<JLB_ACT_SILU, GRAD>(P, taddr, turn, first, row0, nj, ib, bias, (__nv_bfloat16 *)out); break;
                    case JLB_ACT_GELU: store_tile<JLB_ACT_GELU, GRAD>(P, taddr, turn, first, row0, nj, ib, bias, (__nv_bfloat16 *)out); break;
                    default: store_tile<JLB_ACT_NONE, GRAD>(P, taddr, turn, first, row0, nj, ib, bias, (__nv_bfloat16 *)out);
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(te0 + (uint32_t)buf * 8u);
            buf ^= 1;
        }
    } else if (warp == kFindWarp) {
        // ------------------------------------------------------------- tiles
        Walk<GRAD> walk;
        walk.init(P);
        int slot = 0, tk = 0;
        uint32_t ph = 1u, tph = 0u;
        for (int t = pair;;) {
            Tile T;
            const bool have = walk.find(P, t, T);
            if (!tc_wait_warp(smem_u32(&ctl->sempty[slot]), ph, abort_flag)) break;
            if (lane == 0) {
                if (!have) T.bn = 0;
                ctl->ring[slot] = T;
                mbar_arrive_count(smem_u32(&ctl->sfull[slot]), 1);
            }
            if (++slot == kTileRing) { slot = 0; ph ^= 1u; }
            if (!have) break;
            if (!P.counter) {
                t += pairs;
                continue;
            }
            // the next number, drawn by the leader and sent to the other CTA,
            // which reports each ticket's place free again (groups without
            // rows let one CTA's roles run ahead of the other's)
            if (rank == 0) {
                if (!tc_wait_warp(smem_u32(&ctl->tack[tk]), tph ^ 1u, abort_flag)) break;
                if (lane == 0) {
                    t = pairs + atomicAdd(P.counter, 1);
                    store_remote(map_rank(smem_u32(&ctl->ticket[tk]), 1), (uint32_t)t, map_rank(smem_u32(&ctl->tbar[tk]), 1));
                }
                t = __shfl_sync(0xffffffffu, t, 0);
            } else {
                __syncwarp();
                mbar_expect_tx(smem_u32(&ctl->tbar[tk]), 4);
                if (!tc_wait_warp(smem_u32(&ctl->tbar[tk]), tph, abort_flag)) break;
                t = *(volatile int *)&ctl->ticket[tk];
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(map_rank(smem_u32(&ctl->tack[tk]), 0));
            }
            if (++tk == kTickets) { tk = 0; tph ^= 1u; }
        }
        // the other CTA's reports of the last tickets have arrived
        if (rank == 0 && P.counter)
            for (int b = 0; b < kTickets; ++b) {
                if (!tc_wait_warp(smem_u32(&ctl->tack[tk]), tph ^ 1u, abort_flag)) break;
                if (++tk == kTickets) { tk = 0; tph ^= 1u; }
            }
    } else if (warp < kLoadWarp + kLoaders / 32) {
        // ------------------------------------------------------ loader warps
        // Loader warp w of the CTA copies rows w*4 + 16*n + lane/8 of a stage,
        // 8 lanes a 128-byte piece; each thread's arrival on the CTA's rows
        // barrier follows its copies' completion by itself, so every stage of
        // the ring can have copies in flight.
        const int lw = warp - kLoadWarp, sub = lane / 8, c8 = lane % 8;
        // rows r = lw*4 + sub + 16*n of a box: r % 8, and so the swizzle, is the same for all n
        const uint32_t at0 = (uint32_t)(lw * 4 + sub) * 128u + (uint32_t)((c8 ^ ((lw * 4 + sub) & 7)) * 16);
        int stage = 0;
        uint32_t pe = 1u, pgo = 0u;
        bool ok = true, bad = false;
        TileReader tiles;
        Tile T;
        bool more = tiles.next(ctl, T, abort_flag);
        int at[8];                                 // product: this lane's row indices of the tile to come
        auto fetch = [&](const Tile &Q) {
            const int b0 = Q.lo + Q.j0 + (int)rank * (Q.bn / 2);
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const int r = lw * 4 + n * 16 + sub;
                at[n] = r < Q.bn / 2 && b0 + r < Q.hi ? __ldg(P.rows + b0 + r) : INT_MIN;
            }
        };
        if (!GRAD && !F32 && more) fetch(T);
        while (ok && more) {
            Tile N;
            const int bh = T.bn / 2, nb = T.bn / 128;
            if (!GRAD && !F32) {
                // the (at most 8) rows of B this lane copies 16 bytes of
                const __nv_bfloat16 *row[8];
                uint32_t some = 0;
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    row[n] = P.gb;
                    if (at[n] == INT_MIN) continue;          // no row of the tile
                    const int64_t s = (int64_t)at[n] - P.base;
                    if (s >= 0 && s < P.glimit) {
                        row[n] = P.gb + s * P.ldb_ + c8 * 8;
                        some |= 1u << n;
                    } else {
                        bad = true;
                    }
                }
                const int rows = (bh - lw * 4 + 15) / 16;       // bh is a multiple of 16: all lanes alike
                for (int kb = T.kb0; kb < T.kb1; ++kb) {
                    if (!tc_wait_warp(smem_u32(&ctl->empty[stage]), pe, abort_flag)) { ok = false; break; }
                    const uint32_t dst = tiles_u32 + (uint32_t)stage * stage_bytes + kABytes + at0;
                    const uint32_t bytes = bytes_at((int64_t)kb * 64 + c8 * 8, P.Kc);
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        const uint32_t q = some >> n & 1u ? bytes : 0u;
                        if (n < rows) copy16(dst + (uint32_t)n * 2048u, q ? row[n] + kb * 64 : P.gb, q);
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&ctl->rows[stage]))
                                 : "memory");
                    if (++stage == P.stages) { stage = 0; pe ^= 1u; }
                    // the next tile's row indices, while this one's copies run
                    if (kb - T.kb0 == min(2, T.kb1 - T.kb0 - 1)) {
                        more = tiles.next(ctl, N, abort_flag);
                        if (more) fetch(N);
                    }
                }
                if (T.kb0 == T.kb1) {
                    more = tiles.next(ctl, N, abort_flag);
                    if (more) fetch(N);
                }
                T = N;
                continue;
            }
            // gradient: zeros over the rows of a group's last step that are not
            // its own; this lane has rows lw*4 + sub + 16*n of every box
            for (int k = T.kb0 * kPlanes; k < T.kb1 * kPlanes; ++k) {
                const int left = T.hi - T.lo - k / kPlanes * 64;
                if (left < 64) {
                    if (!tc_wait_warp(smem_u32(&ctl->go[stage]), pgo >> stage & 1u, abort_flag)) { ok = false; break; }
                    pgo ^= 1u << stage;           // a bit a stage: its next use comes after its release
                    const uint32_t dst = tiles_u32 + (uint32_t)stage * stage_bytes + at0;
#pragma unroll
                    for (int n = 0; n < 4; ++n)
                        if (lw * 4 + sub + 16 * n >= left)
                            for (int x = 0; x < 2 + nb; ++x)
                                zero16(dst + (uint32_t)x * kBox + (uint32_t)n * 2048u);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    mbar_arrive_count(smem_u32(&ctl->rows[stage]), 1);
                }
                if (++stage == P.stages) stage = 0;
            }
            more = tiles.next(ctl, T, abort_flag);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (bad) dev_error(DEV_ERR_BOUNDS);
    } else {
        // ------------------------------------------------- the loaders' report
        // A stage whose rows are in place: the copies (generic proxy) are made
        // visible to the tensor cores' reads (async proxy), then the leader's
        // barrier gets this CTA's arrival.
        const uint32_t full0 = map_rank(smem_u32(&ctl->full[0]), 0);
        int stage = 0;
        uint32_t pr = 0;                          // the phase of each stage's rows barrier, a bit each
        bool ok = true;
        TileReader tiles;
        Tile T;
        while (ok && tiles.next(ctl, T, abort_flag)) {
            for (int k = T.kb0 * kPlanes; k < T.kb1 * kPlanes; ++k) {
                if (!GRAD || T.hi - T.lo - k / kPlanes * 64 < 64) {
                    if (!tc_wait_warp(smem_u32(&ctl->rows[stage]), (pr >> stage) & 1u, abort_flag)) { ok = false; break; }
                    pr ^= 1u << stage;
                    if (lane == 0) {
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        mbar_arrive_cluster(full0 + (uint32_t)stage * 8u);
                    }
                    __syncwarp();
                }
                if (++stage == P.stages) stage = 0;
            }
        }
    }

    __syncthreads();
    // every copy has landed and every product is done before shared memory and
    // TMEM go (after an abort some may still be on their way)
    if (threadIdx.x == 0) {
        tc_drain(smem_u32(&ctl->done), 0);
        for (int s = 0; s < P.stages; ++s)
            if (ctl->tails >> s & 1u) tc_drain(smem_u32(&ctl->go[s]), (ctl->tail_phase >> s & 1u) ^ 1u);
        if (rank == 0 && ctl->abort)
            for (uint32_t s = 0; s < (uint32_t)P.stages && s < ctl->fills; ++s)
                tc_drain(smem_u32(&ctl->full[s]), ((ctl->fills - 1 - s) / (uint32_t)P.stages) & 1u);
    }
    __syncthreads();
    // neither CTA's shared memory goes before the other is done.  Arrivals on
    // the other CTA's barriers have been waited for there (empty, tfull and done
    // of commits; full, tempty and tack on the leader; tbar), unless a wait
    // gave up: the role at the other end then gives up too, and its CTA's barrier
    // is one that its arrivals come before.
    if (ctl->abort) cluster_sync_released();
    else cluster_sync_relaxed();
    if (warp == 1) {
        fence_after();
        dealloc_pair(tmem, 512);
    }
}

// The split tiles: adds their parts in order and applies the epilogue.  CTA
// (x, y): kFinish columns of the y-th split tile, one lane a thread; four
// parts of them are loaded before any is added.  Launched
// while product_tc runs; the wait ends when that grid is complete.
constexpr int kFinish = 4;
template <bool GRAD, typename T_>
__global__ void __launch_bounds__(256) finish_tc(const __grid_constant__ TcArgs P) {
    __shared__ Tile ts;
    __shared__ int ns;
    if (threadIdx.x < kWarp) {
        Walk<GRAD> walk;
        walk.init(P);
        Tile T;
        const bool have = walk.splits > 1 && walk.find(P, walk.full + blockIdx.y * walk.splits, T);
        if (threadIdx.x == 0) {
            ns = have ? walk.splits : 0;
            if (have) ts = T;
        }
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (ns == 0) return;
    const Tile T = ts;
    const int nj = GRAD ? (int)min((int64_t)T.bn, P.J - T.j0) : min(T.bn, T.hi - T.lo - T.j0);
    const int c0 = blockIdx.x * kFinish;
    const int64_t i = (int64_t)T.i0 + threadIdx.x, item = (int64_t)256 * P.bn_max;
    if (i >= P.I || c0 >= nj) return;
    const float *part = P.part + (int64_t)blockIdx.y * ns * item + threadIdx.x;
    const float bias = !GRAD && P.bias ? to_f32(((const T_ *)P.bias)[T.e * P.ldb + i]) : 0.0f;
    T_ *out = (T_ *)P.out + (GRAD ? T.e * P.out_stride : 0) + i;
    const int64_t row0 = GRAD ? T.j0 : (int64_t)T.lo + T.j0;
    float sum[kFinish] = {};
    for (int s0 = 0; s0 < ns; s0 += 4) {
        float v[4][kFinish];
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int c = 0; c < kFinish; ++c)
                v[q][c] = s0 + q < ns && c0 + c < nj ? part[(s0 + q) * item + (int64_t)(c0 + c) * 256] : 0.0f;
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int c = 0; c < kFinish; ++c) sum[c] += v[q][c];
    }
#pragma unroll
    for (int x = 0; x < kFinish; ++x) {
        const int c = c0 + x;
        if (c >= nj) break;
        float v = sum[x];
        const int64_t r = row0 + c;
        if (!GRAD) {
            v += bias;
            if (P.z) ((T_ *)P.z)[r * P.ldz + i] = from_f32<T_>(v);
            v = act_value<T_>(v, P.act);
            if (P.res) v = add_rn(v, to_f32(((const T_ *)P.res)[r * P.ldr + i]));
        }
        out[r * P.ldo] = from_f32<T_>(v);
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

static bool encode(CUtensorMap *m, const void *p, int rank, const cuuint64_t *dims, const cuuint64_t *strides,
                   const cuuint32_t *box) {
    auto fn = encode_fn();
    const cuuint32_t es[4] = {1, 1, 1, 1};
    return fn && fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void *>(p), dims, strides, box, es,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// rows x cols (x experts) of bf16 as {cols, rows[, experts]}, box {64, box_rows}.
static bool make_map(CUtensorMap *m, const void *p, int64_t cols, int64_t rows, int64_t ld, int64_t experts,
                     int64_t stride, int box_rows) {
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)experts};
    const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
    return encode(m, p, experts > 0 ? 3 : 2, dims, strides, box);
}

// The same matrices as {64, rows, cols / 64[, experts]}, so that one copy of
// box {64, 64, 2} brings two neighbouring 64-column boxes, stacked.  Only for
// cols a multiple of 64: the last box would otherwise leave its row.
static bool make_pair_map(CUtensorMap *m, const void *p, int64_t cols, int64_t rows, int64_t ld, int64_t experts,
                          int64_t stride) {
    if (cols % 64) return false;
    const cuuint64_t dims[4] = {64, (cuuint64_t)rows, (cuuint64_t)(cols / 64), (cuuint64_t)experts};
    const cuuint64_t strides[3] = {(cuuint64_t)ld * 2, 128, (cuuint64_t)stride * 2};
    const cuuint32_t box[4] = {64, 64, 2, 1};
    return encode(m, p, experts > 0 ? 4 : 3, dims, strides, box);
}

static bool tma_matrix(const void *p, int64_t ld) { return aligned16(p) && ld % 8 == 0; }

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

// Columns of the instruction a call needs at most, and how its tiles are
// split: tiles is their number (product: an upper bound when rowptr decides).
constexpr size_t kCounterBytes = 256;                   // the workspace's first bytes: the tile counter
struct TcPlan {
    int bn_max, pairs, max_splits, full, splits;
    bool finish, dynamic;
    int rest;                      // split tiles, at most
    size_t part_bytes;
};
static TcPlan tc_plan(int bn_max, int64_t tiles, bool exact, bool ragged, int64_t steps) {
    TcPlan p{bn_max, device_sms() / 2, 1, INT32_MAX, 1, false, false, 0, 0};
    if (tiles > INT32_MAX / 2) return p;           // the launch refuses
    // at least four steps a part; and finish_tc's launch is worth it only when
    // a partly filled last round can be a sixth of the work
    int64_t most = steps / 4 < 64 ? steps / 4 : 64;
    if (tiles >= 6 * (int64_t)p.pairs) most = 1;
    if (exact) {
        split_schedule((int)tiles, p.pairs, (int)most, p.full, p.splits);
        p.finish = p.splits > 1;
        p.rest = (int)tiles - p.full;
    } else if (most > 1) {
        p.max_splits = (int)most;
        p.finish = true;
        p.rest = p.pairs / 2;                      // a split tile has two parts at least
    }
    if (p.finish) p.part_bytes = (size_t)p.pairs * 256 * bn_max * 4;
    else if (tiles < p.pairs) p.pairs = (int)tiles;
    // handed out where tiles differ in cost and two rounds or more of them hide
    // the counter's clearing (3.5 us): gradients of 8192 rows over 16 experts 375
    // -> 365 us, a 32,044-row prefill 558 -> 544; decode steps' tiles are alike
    p.dynamic = ragged && tiles > 2 * p.pairs;
    return p;
}

template <bool A_MN, bool GRAD, typename T_>
static int launch_tc(cudaStream_t st, const CUtensorMap &a, const CUtensorMap &b, const CUtensorMap &big,
                     const CUtensorMap &mid, TcArgs &P,
                     const TcPlan &plan, void *ws, bool loaders) {
    const size_t extra = 1024 + kTurnBytes + sizeof(TcCtl);
    const uint32_t stage = stage_size(plan.bn_max);
    P.bn_max = plan.bn_max;
    const int64_t inner = GRAD ? P.S / P.E : P.Kc, tile = (inner > 0 ? inner : 1) * plan.bn_max * 2 * (sizeof(T_) == 4 ? 3 : 1);
    P.jblock = (int)(kL2Block / tile < 4 ? 4 : kL2Block / tile > 64 ? 64 : kL2Block / tile);
    P.pairs = plan.pairs;
    P.max_splits = plan.max_splits;
    P.full = plan.full;
    P.splits = plan.splits;
    P.part = (float *)((char *)ws + kCounterBytes);
    P.counter = plan.dynamic ? (int *)ws : nullptr;
    if (plan.dynamic) JLB_CUDA(cudaMemsetAsync(ws, 0, sizeof(int), st));
    P.stages = (int)((227 * 1024 - extra) / stage);
    if (P.stages > kMaxStages) P.stages = kMaxStages;
    const size_t smem = (size_t)P.stages * stage + extra;
    JLB_CUDA(cudaFuncSetAttribute(product_tc<A_MN, GRAD, T_>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    product_tc<A_MN, GRAD, T_><<<(unsigned)(2 * P.pairs), kTcThreads + (loaders ? kLoaders + kForward : 0), smem, st>>>(a, b, big, mid, P);
    JLB_LAUNCH_CHECK("product_tc");
    if (plan.finish) {
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.gridDim = dim3((unsigned)ceil_div(P.bn_max, kFinish), (unsigned)plan.rest);
        cfg.blockDim = dim3(256);
        cfg.stream = st;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        JLB_CUDA(cudaLaunchKernelEx(&cfg, finish_tc<GRAD, T_>, P));
    }
    return ok();
}

static int widest(int dtype) { return dtype == JLB_F32 ? 128 : 256; }   // F32: sums in registers

static TcPlan plan_product(const Product &p) {
    const int wide = widest(p.dtype), bn = p.S >= wide ? wide : (int)((p.S + 31) / 32 * 32);
    if (!p.rowptr)
        return tc_plan(bn, col_tiles((int)p.S, bn) * ceil_div(p.N, 256), true, false, ceil_div(p.K, 64));
    const int64_t cols = ceil_div(p.S, bn) + (p.E < p.S ? p.E : p.S);
    return tc_plan(bn, cols * ceil_div(p.N, 256), false, p.S >= 64 * p.E, ceil_div(p.K, 64));
}

static TcPlan plan_gradient(const Gradient &g) {
    const int64_t J = g.w_order == JLB_ROW_MAJOR ? g.K : g.N, I = g.w_order == JLB_ROW_MAJOR ? g.N : g.K;
    const int bn = J > 128 ? widest(g.dtype) : 128;
    return tc_plan(bn, g.E * ceil_div(I, 256) * ceil_div(J, bn), true, g.E > 1 && g.S >= 64 * g.E, ceil_div(g.S / g.E, 64));
}

static size_t plan_bytes(const TcPlan &p) { return p.part_bytes || p.dynamic ? kCounterBytes + p.part_bytes : 0; }
size_t tc_product_workspace(const Product &P) { return plan_bytes(plan_product(P)); }
size_t tc_gradient_workspace(const Gradient &G) { return plan_bytes(plan_gradient(G)); }

// Status, or -1 when the driver refuses a tensor map (the caller takes
// another kernel).  F32: p.x and p.w are three bf16 planes each, [3][T][ldx]
// and [3][E] matrices, bias, res, z and y are F32.
int tc_product(cudaStream_t st, const Product &p, void *ws) {
    const int planes = p.dtype == JLB_F32 ? 3 : 1;
    CUtensorMap a, b, big, mid;
    const bool mn = p.w_order == JLB_ROW_MAJOR;
    const int64_t experts = p.E * planes, w_stride = experts > 1 ? p.w_stride : (mn ? p.K : p.N) * p.ldw;
    const bool pair = mn && make_pair_map(&a, p.w, p.N, p.K, p.ldw, experts, w_stride);
    if (!pair && !(mn ? make_map(&a, p.w, p.N, p.K, p.ldw, experts, w_stride, 64)
                      : make_map(&a, p.w, p.K, p.N, p.ldw, experts, w_stride, 128)))
        return -1;
    if (!make_map(&b, p.x, p.K, p.T * planes, p.ldx, 0, 0, 32) ||
        !make_map(&mid, p.x, p.K, p.T * planes, p.ldx, 0, 0, 64) ||
        !make_map(&big, p.x, p.K, p.T * planes, p.ldx, 0, 0, 128))
        return -1;
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
    P.a_pair = pair;
    P.pa = (int)p.E;
    P.pb = (int)p.T;
    P.gb = (const __nv_bfloat16 *)p.x;
    P.ldb_ = p.ldx;
    P.bias = p.bias;
    P.ldb = p.ldb;
    P.res = p.res;
    P.ldr = p.ldr;
    P.z = p.z;
    P.ldz = p.ldz;
    P.out = p.y;
    P.ldo = p.ldy;
    P.vec = tma_matrix(p.y, p.ldy) && (!p.z || tma_matrix(p.z, p.ldz));
    const TcPlan plan = plan_product(p);
    if (plan.pairs < 1 || (p.rowptr ? p.E : 1) * ceil_div(p.N, 256) * ceil_div(p.S, 32) > INT32_MAX / 2) return -1;
    if (p.dtype == JLB_F32)
        return mn ? launch_tc<true, false, float>(st, a, b, big, mid, P, plan, ws, false)
                  : launch_tc<false, false, float>(st, a, b, big, mid, P, plan, ws, false);
    return mn ? launch_tc<true, false, __nv_bfloat16>(st, a, b, big, mid, P, plan, ws, p.rows)
              : launch_tc<false, false, __nv_bfloat16>(st, a, b, big, mid, P, plan, ws, p.rows);
}

int tc_gradient(cudaStream_t st, const Gradient &g, void *ws) {
    // dw row-major: lanes = columns n (dz), columns = k (x); column-major: exchanged
    const int planes = g.dtype == JLB_F32 ? 3 : 1;
    const bool row = g.w_order == JLB_ROW_MAJOR;
    const void *ap = row ? g.dz : g.x, *bp = row ? g.x : g.dz;
    const int64_t ac = row ? g.N : g.K, ar = row ? g.S : g.T, lda = row ? g.lddz : g.ldx;
    const int64_t bc = row ? g.K : g.N, br = row ? g.T : g.S, ldb = row ? g.ldx : g.lddz;
    CUtensorMap a, b, big, mid;
    const bool a_pair = make_pair_map(&a, ap, ac, ar * planes, lda, 0, 0),
               b_pair = make_pair_map(&big, bp, bc, br * planes, ldb, 0, 0);
    if ((!a_pair && !make_map(&a, ap, ac, ar * planes, lda, 0, 0, 64)) || !make_map(&b, bp, bc, br * planes, ldb, 0, 0, 64))
        return -1;
    if (!b_pair) big = b;
    mid = b;
    TcArgs P{};
    P.base = g.base;
    P.E = g.E;
    P.S = g.S;
    P.I = ac;
    P.J = bc;
    P.a_pair = a_pair;
    P.b_pair = b_pair;
    P.pa = (int)ar;
    P.pb = (int)br;
    P.rowptr = g.rowptr;
    P.vec = tma_matrix(g.dw, g.lddw) && (g.E == 1 || g.dw_stride % 8 == 0);
    P.out = g.dw;
    P.ldo = g.lddw;
    P.out_stride = g.dw_stride;
    if (P.E * ceil_div(P.I, 256) * ceil_div(P.J, 128) > INT32_MAX / 2) return -1;
    return g.dtype == JLB_F32 ? launch_tc<true, true, float>(st, a, b, big, mid, P, plan_gradient(g), ws, true)
                              : launch_tc<true, true, __nv_bfloat16>(st, a, b, big, mid, P, plan_gradient(g), ws, true);
}

}  // namespace emm
}  // namespace jlb
