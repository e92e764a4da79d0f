// expert_mm.cu -- products grouped by expert over ragged row ranges, with
// bias, activation and residual in the epilogue, and their gradients.  The
// dense product is the same call with one group.
//
// This file holds the entry points, the copies that make operands fit the
// tensor path (aligned rows of bf16, planes of F32) and the kernels without
// tensor cores, for shapes the tensor path does not take.
#include "expert_mm.cuh"

#include <new>

namespace jlb {

JLB_DEFINE_DEV_ERROR(emm)

namespace emm {

// ------------------------------------------------ tiled product, FFMA
// out (M x N) = A (M x Kc) B (Kc x N) on 128 x 128 tiles, 16 of the inner
// dimension a step, 256 threads with 8 x 8 sums each in fp32 registers.  An
// operand is "k-contiguous" when neighbouring inner indices are neighbours in
// memory, else its outer index is.
constexpr int kTile = 128, kStep = 16, kSimtThreads = 256;
constexpr int kPitch = kTile + 4;

// Element source: outer index o (row of A or column of B), inner index i.
template <typename T>
struct Operand {
    const T *p;
    int64_t ld;
    bool k_contig;
    const int32_t *gather;   // maps the row index of the stored matrix, or null
    int gbase;
    int64_t glimit;          // rows the gathered matrix has
    int row0;                // added to the row index of the stored matrix
    // The stored matrix's row is the outer index when k_contig, else the inner.
    __device__ __forceinline__ const T *row_ptr(int64_t r, bool &bad) const {
        r += row0;
        if (gather) {
            r = (int64_t)__ldg(gather + r) - gbase;
            if (r < 0 || r >= glimit) {
                bad = true;
                return nullptr;
            }
        }
        return p + r * ld;
    }
};

// Loads a kTile x kStep tile (outer x inner) into dst[inner][outer]; zeros
// outside omax x imax.
template <typename T>
__device__ __forceinline__ void load_tile(const Operand<T> &op, int64_t o0, int64_t omax,
                                          int64_t i0, int64_t imax, float (*dst)[kPitch]) {
    const int tid = threadIdx.x;
    bool bad = false;
    if (op.k_contig) {
        const int o = tid % kTile, ih = (tid / kTile) * 8;
        const bool in = o0 + o < omax;
        const T *r = in ? op.row_ptr(o0 + o, bad) : nullptr;
#pragma unroll
        for (int c = 0; c < 8; ++c)
            dst[ih + c][o] = r && i0 + ih + c < imax ? to_f32(r[i0 + ih + c]) : 0.0f;
    } else {
        const int i = tid / 16, o8 = (tid % 16) * 8;
        const bool in = i0 + i < imax;
        const T *r = in ? op.row_ptr(i0 + i, bad) : nullptr;
#pragma unroll
        for (int c = 0; c < 8; ++c)
            dst[i][o8 + c] = r && o0 + o8 + c < omax ? to_f32(r[o0 + o8 + c]) : 0.0f;
    }
    if (bad) dev_error(DEV_ERR_BOUNDS);
}

template <typename T>
__device__ __forceinline__ void tile_product(const Operand<T> &A, int64_t m0, int64_t mmax,
                                             const Operand<T> &B, int64_t n0, int64_t nmax,
                                             int64_t kmax, float (&acc)[8][8]) {
    __shared__ __align__(16) float sa[kStep][kPitch];
    __shared__ __align__(16) float sb[kStep][kPitch];
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = 0.0f;
    for (int64_t k0 = 0; k0 < kmax; k0 += kStep) {
        load_tile(A, m0, mmax, k0, kmax, sa);
        load_tile(B, n0, nmax, k0, kmax, sb);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kStep; ++k) {
            float a[8], b[8];
            *reinterpret_cast<float4 *>(a) = *reinterpret_cast<const float4 *>(&sa[k][ty * 4]);
            *reinterpret_cast<float4 *>(a + 4) = *reinterpret_cast<const float4 *>(&sa[k][64 + ty * 4]);
            *reinterpret_cast<float4 *>(b) = *reinterpret_cast<const float4 *>(&sb[k][tx * 4]);
            *reinterpret_cast<float4 *>(b + 4) = *reinterpret_cast<const float4 *>(&sb[k][64 + tx * 4]);
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
}

__device__ __forceinline__ int tile_index(int t, int i) { return (i < 4 ? 0 : 64) + t * 4 + (i & 3); }

// Grid extents y and z hold 65,535 CTAs each: numbers up to n lie in y and, past
// that, in z (a loop in the kernel instead made act_backward 28 % slower).
static dim3 in_yz(int64_t x, int64_t n) {
    const int64_t y = n < 65535 ? n : 65535;
    return dim3((unsigned)x, (unsigned)y, (unsigned)(y ? ceil_div(n, y) : 1));
}
__device__ __forceinline__ int64_t at_yz() { return (int64_t)blockIdx.z * gridDim.y + blockIdx.y; }

// The group and first row of row tile `want`, tiles of `size` rows numbered
// group by group; e = -1 past the last.  Warp 0 scans 32 groups at a time.
struct Found {
    int e, lo, hi, row0;
};
__device__ void find_row_tile(const int32_t *rowptr, int base, int64_t S, int64_t E, int size,
                              int64_t want, Found *out) {
    if (threadIdx.x >= kWarp) return;
    const int lane = threadIdx.x;
    int64_t before = 0;
    if (lane == 0) out->e = -1;
    for (int64_t e0 = 0; e0 < E; e0 += kWarp) {
        int lo = 0, hi = 0;
        if (e0 + lane < E) group_rows(rowptr, base, S, e0 + lane, lo, hi);
        const int tiles = (int)ceil_div(hi - lo, size);
        int inc = tiles;
#pragma unroll
        for (int o = 1; o < kWarp; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        const int64_t first = before + inc - tiles;
        if (want >= first && want < first + tiles)
            *out = Found{(int)(e0 + lane), lo, hi, lo + (int)(want - first) * size};
        before += __shfl_sync(0xffffffffu, inc, 31);
        if (want < before) break;
    }
}

template <typename T>
__global__ void __launch_bounds__(kSimtThreads) product_simt(const Product P) {
    __shared__ Found f;
    const int64_t tile = at_yz(), tiles = (int64_t)gridDim.z * gridDim.y;
    find_row_tile(P.rowptr, P.base, P.S, P.E, kTile, tile, &f);
    if (blockIdx.x == 0 && P.rowptr) {
        for (int64_t e = tile * kSimtThreads + threadIdx.x; e < P.E; e += tiles * kSimtThreads)
            if (group_bad(P.rowptr, P.base, P.S, e)) dev_error(DEV_ERR_BOUNDS);
    }
    // rows of no group are zero
    if (P.rowptr) {
        int lo, hi;
        group_rows(P.rowptr, P.base, P.S, P.E - 1, lo, hi);
        for (int64_t r = hi + tile; r < P.S; r += tiles)
            for (int64_t c = (int64_t)blockIdx.x * kSimtThreads + threadIdx.x; c < P.N;
                 c += (int64_t)gridDim.x * kSimtThreads) {
                ((T *)P.y)[r * P.ldy + c] = from_f32<T>(0.0f);
                if (P.z) ((T *)P.z)[r * P.ldz + c] = from_f32<T>(0.0f);
            }
    }
    __syncthreads();
    if (f.e < 0) return;
    const int64_t n0 = (int64_t)blockIdx.x * kTile;
    Operand<T> A{(const T *)P.x, P.ldx, true, P.rows, P.base, P.T, f.row0};
    Operand<T> B{(const T *)P.w + f.e * P.w_stride, P.ldw, P.w_order == JLB_COL_MAJOR, nullptr, 0, 0, 0};
    float acc[8][8];
    tile_product<T>(A, 0, f.hi - f.row0, B, n0, P.N, P.K, acc);
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = f.row0 + tile_index(ty, i);
        if (r >= f.hi) continue;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t n = n0 + tile_index(tx, j);
            if (n >= P.N) continue;
            float v = acc[i][j];
            if (P.bias) v += to_f32(((const T *)P.bias)[f.e * P.ldb + n]);
            if (P.z) ((T *)P.z)[r * P.ldz + n] = from_f32<T>(v);
            v = act_value<T>(v, P.act);
            if (P.res) v = add_rn(v, to_f32(((const T *)P.res)[r * P.ldr + n]));
            ((T *)P.y)[r * P.ldy + n] = from_f32<T>(v);
        }
    }
}

// dw[e] on 128 x 128 tiles; the inner dimension is the group's rows.  A
// column-major dw is computed as its transpose, the operands swapped.
template <typename T>
__global__ void __launch_bounds__(kSimtThreads) gradient_simt(const Gradient G) {
    const bool col = G.w_order == JLB_COL_MAJOR;
    const int64_t M = col ? G.N : G.K, N = col ? G.K : G.N, n0 = (int64_t)blockIdx.x * kTile;
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    for (int64_t e = blockIdx.z; e < G.E; e += gridDim.z) {
        int lo, hi;
        group_rows(G.rowptr, G.base, G.S, e, lo, hi);
        if (group_bad(G.rowptr, G.base, G.S, e) && threadIdx.x == 0) dev_error(DEV_ERR_BOUNDS);
        Operand<T> X{(const T *)G.x, G.ldx, false, G.rows, G.base, G.T, lo};
        Operand<T> D{(const T *)G.dz, G.lddz, false, nullptr, 0, 0, lo};
        T *out = (T *)G.dw + e * G.dw_stride;
        for (int64_t m0 = (int64_t)blockIdx.y * kTile; m0 < M; m0 += (int64_t)gridDim.y * kTile) {
            float acc[8][8];
            tile_product<T>(col ? D : X, m0, M, col ? X : D, n0, N, hi - lo, acc);
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int64_t r = m0 + tile_index(ty, i), c = n0 + tile_index(tx, j);
                    if (r < M && c < N) out[r * G.lddw + c] = from_f32<T>(acc[i][j]);
                }
        }
    }
}

// ------------------------------------------------- activation's gradient
// dz = dy * act'(z), and the column sums of each group's dz (the bias's
// gradient) over kSumRows rows a CTA: 32 threads of V columns (16 bytes, or
// one where the layout is not aligned) x 8 row lanes, four rows' loads on
// their way at a time.  Sums of unrounded products in fp32: a lane's rows,
// then the 8 lanes in order; sum_parts adds a group's CTAs in order.  Bound by
// HBM.  Row ranges that overlap (rowptr running backwards) have more tiles than
// rows allow: the ones past the grid are left out, in sum_parts too, and
// reported.
constexpr int kSumRows = 128;
template <typename T, int V>
struct Values {                    // as they lie in memory, until they are used
    uint4 q;
    T one;
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (V == 1) one = *p;
        else q = *reinterpret_cast<const uint4 *>(p);
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (V == 1) return to_f32(one);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
        return sizeof(T) == 4 ? __uint_as_float(w[i % 4])
                              : __uint_as_float(i % 2 ? w[i / 2 % 4] & 0xffff0000u : w[i / 2 % 4] << 16);
    }
};
template <typename T, int V>
__device__ __forceinline__ void store_v(T *p, const float (&v)[V]) {
    if constexpr (V == 1) {
        *p = from_f32<T>(v[0]);
    } else {
        __align__(16) T o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = from_f32<T>(v[i]);
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(o);
    }
}

template <typename T, int V, int ACT>
__device__ __forceinline__ void act_rows(int lo, int hi, int64_t c, const T *__restrict__ dy, int64_t lddy,
                                         const T *__restrict__ z, int64_t ldz, T *__restrict__ dz, int64_t lddz,
                                         float (&sum)[V]) {
    constexpr int U = 4;
    for (int r0 = lo + threadIdx.x / 32; r0 < hi; r0 += 8 * U) {
        Values<T, V> d[U], q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t r = r0 + 8 * u;
            if (r < hi) {
                d[u].load(dy + r * lddy + c);
                if (ACT != JLB_ACT_NONE) q[u].load(z + r * ldz + c);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t r = r0 + 8 * u;
            if (r >= hi) break;
            float v[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[i] = d[u].get(i);
                if (ACT != JLB_ACT_NONE) v[i] *= act_slope<T>(q[u].get(i), ACT);
                sum[i] += v[i];
            }
            if (dz) store_v<T, V>(dz + r * lddz + c, v);
        }
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(256, 4)
act_backward(int64_t tiles, int64_t E, int64_t S, int64_t N, int base, const int32_t *__restrict__ rowptr, int act,
             const T *__restrict__ dy, int64_t lddy, const T *__restrict__ z, int64_t ldz,
             T *__restrict__ dz, int64_t lddz, float *__restrict__ part) {
    __shared__ Found f;
    __shared__ float red[8][32 * V];
    const int64_t tile = at_yz();
    if (tile >= tiles) return;                     // part has no place for it
    find_row_tile(rowptr, base, S, E, kSumRows, tile, &f);
    if (blockIdx.x == 0)
        for (int64_t e = tile * 256 + threadIdx.x; e < E; e += tiles * 256)
            if (group_bad(rowptr, base, S, e)) dev_error(DEV_ERR_BOUNDS);
    __syncthreads();
    if (f.e < 0) return;
    const int cx = threadIdx.x % 32;
    const int64_t c = ((int64_t)blockIdx.x * 32 + cx) * V;
    const int hi = min(f.hi, f.row0 + kSumRows);
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.0f;
    if (c < N) {
        switch (act) {
            case JLB_ACT_RELU: act_rows<T, V, JLB_ACT_RELU>(f.row0, hi, c, dy, lddy, z, ldz, dz, lddz, sum); break;
            case JLB_ACT_SILU: act_rows<T, V, JLB_ACT_SILU>(f.row0, hi, c, dy, lddy, z, ldz, dz, lddz, sum); break;
            case JLB_ACT_GELU: act_rows<T, V, JLB_ACT_GELU>(f.row0, hi, c, dy, lddy, z, ldz, dz, lddz, sum); break;
            default: act_rows<T, V, JLB_ACT_NONE>(f.row0, hi, c, dy, lddy, z, ldz, dz, lddz, sum);
        }
    }
    if (!part) return;
#pragma unroll
    for (int i = 0; i < V; ++i) red[threadIdx.x / 32][cx * V + i] = sum[i];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * V; i += 256) {
        const int64_t col = (int64_t)blockIdx.x * 32 * V + i;
        if (col >= N) continue;
        float s = red[0][i];
#pragma unroll
        for (int q = 1; q < 8; ++q) s += red[q][i];
        part[tile * N + col] = s;
    }
}

// part holds `parts` rows of N.
template <typename T>
__global__ void __launch_bounds__(256)
sum_parts(int64_t E, int64_t S, int64_t N, int base, const int32_t *__restrict__ rowptr,
          const float *__restrict__ part, int64_t parts, T *__restrict__ db, int64_t lddb) {
    const int64_t e = at_yz();
    __shared__ int64_t first_s;
    __shared__ int count_s;
    if (e >= E) return;
    if (threadIdx.x < kWarp) {                 // the group's parts: after those of the groups before
        int64_t first = 0;
        for (int64_t i = threadIdx.x; i < e; i += kWarp) {
            int lo, hi;
            group_rows(rowptr, base, S, i, lo, hi);
            first += ceil_div(hi - lo, kSumRows);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) first += __shfl_xor_sync(0xffffffffu, first, o);
        if (threadIdx.x == 0) {
            int lo, hi;
            group_rows(rowptr, base, S, e, lo, hi);
            const int64_t left = parts > first ? parts - first : 0, count = ceil_div(hi - lo, kSumRows);
            first_s = first;
            count_s = (int)(count < left ? count : left);
        }
    }
    __syncthreads();
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= N) return;
    float s = 0.0f;
#pragma unroll 8
    for (int i = 0; i < count_s; ++i) s += part[(first_s + i) * N + c];
    db[e * lddb + c] = from_f32<T>(s);
}

template <typename T>
static int launch_act(cudaStream_t st, int64_t tiles, int64_t E, int64_t S, int64_t N, int base, const int32_t *rowptr,
                      int act, const void *dy, int64_t lddy, const void *z, int64_t ldz, void *dz, int64_t lddz,
                      float *part) {
    constexpr int V = 16 / (int)sizeof(T);
    const bool vec = N % V == 0 && lddy % V == 0 && aligned16(dy) && (!z || (ldz % V == 0 && aligned16(z))) &&
                     (!dz || (lddz % V == 0 && aligned16(dz)));
    const dim3 grid = in_yz(ceil_div(N, vec ? 32 * V : 32), tiles);
    if (vec)
        act_backward<T, V><<<grid, 256, 0, st>>>(tiles, E, S, N, base, rowptr, act, (const T *)dy, lddy, (const T *)z, ldz,
                                                 (T *)dz, lddz, part);
    else
        act_backward<T, 1><<<grid, 256, 0, st>>>(tiles, E, S, N, base, rowptr, act, (const T *)dy, lddy, (const T *)z, ldz,
                                                 (T *)dz, lddz, part);
    JLB_LAUNCH_CHECK("act_backward");
    return JLB_OK;
}

static int64_t row_tiles_bound(int64_t E, int64_t S, bool ragged, int size) {
    return ceil_div(S, size) + (ragged ? (E < S ? E : S) : 0);
}

static int check_types(int dtype, int idx_base) {
    if (dtype != JLB_F32 && dtype != JLB_BF16)
        return fail(JLB_ERR_UNSUPPORTED_VALUE_TYPE, "grouped products run on F32 and BF16 values");
    if (idx_base != 0 && idx_base != 1) return fail(JLB_ERR_INVALID_ARGUMENT, "idx_base must be 0 or 1");
    return JLB_OK;
}

static int check_extents(int64_t E, int64_t S, int64_t T, int64_t K, int64_t N,
                         const int32_t *rowptr, const int32_t *rows) {
    if (E < 0 || S < 0 || T < 0 || K < 0 || N < 0)
        return fail(JLB_ERR_INCOMPATIBLE_EXTENTS, "negative extent");
    if (!rowptr && E != 1)
        return fail(JLB_ERR_INVALID_ARGUMENT, "no row pointer: only one group has all the rows");
    if (!rows && S != T && S > 0)                 // an empty index buffer may have no address
        return fail(JLB_ERR_INCOMPATIBLE_EXTENTS, "x has %lld rows, the result %lld", (long long)T,
                    (long long)S);
    if (S > (int64_t)INT32_MAX - 1024 || T > (int64_t)INT32_MAX - 1024 ||
        E > (int64_t)INT32_MAX - 1024 || K > (int64_t)INT32_MAX - 1024 || N > (int64_t)INT32_MAX - 1024)
        return fail(JLB_ERR_UNSUPPORTED_INDEX_TYPE, "extent exceeds Int32 positions");
    return JLB_OK;
}

static int check_weight(int order, int64_t E, int64_t K, int64_t N, int64_t ldw, int64_t stride) {
    if (order != JLB_ROW_MAJOR && order != JLB_COL_MAJOR)
        return fail(JLB_ERR_INVALID_ARGUMENT, "weight order must be row- or column-major");
    if (ldw < (order == JLB_ROW_MAJOR ? N : K))
        return fail(JLB_ERR_INCOMPATIBLE_EXTENTS, "weight leading dimension too small");
    if (E > 1 && stride < (order == JLB_ROW_MAJOR ? (K > 0 ? (K - 1) * ldw + N : 0)
                                                   : (N > 0 ? (N - 1) * ldw + K : 0)))
        return fail(JLB_ERR_INCOMPATIBLE_EXTENTS, "experts' weights overlap");
    return JLB_OK;
}

static int check_act(int act) {
    return act < JLB_ACT_NONE || act > JLB_ACT_GELU
               ? fail(JLB_ERR_INVALID_ARGUMENT, "unknown activation %d", act)
               : JLB_OK;
}

// ------------------------------------------------- copies for the tensor path
static int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }
static size_t pad256(size_t n) { return (n + 255) / 256 * 256; }
static bool tma_rows(const void *p, int64_t ld) { return aligned16(p) && ld % 8 == 0; }

// Rows of one operand that the tensor path reads from a copy.
struct Copy {
    const void *src;              // experts matrices of rows x cols
    int64_t experts, rows, cols, ld, stride;
    const int32_t *idx;           // source row of each row, or null; an index outside [0, limit): a row of zeros
    int64_t limit;
    const int32_t *live_end;      // rows from *live_end on are of no group and hold nothing
    const int32_t *rowptr;        // matrices whose group has none of the S rows are not read, or null: all are
    int64_t S;
    int base, vec;                // vec: the source's rows are 16-byte aligned
    void *dst;
    int64_t ldd;
    int64_t warps;                // pieces of rows, one a warp at a time
};

// Where piece w of a copy comes from: its row r of the copy and its source
// row, null for a row of zeros.  False: nothing to do.
template <typename T>
__device__ __forceinline__ bool copy_source(const Copy &c, int64_t w, int per_piece, int64_t &r, int64_t &col,
                                            const T *&s, bool &outside) {
    const int64_t pieces = (c.cols + per_piece - 1) / per_piece;
    r = pieces == 1 ? w : w / pieces;
    col = (w - r * pieces) * per_piece;
    const int64_t e = c.experts == 1 ? 0 : r / c.rows;
    int64_t sr = r - e * c.rows;
    if (c.live_end && sr >= (int64_t)__ldg(c.live_end) - c.base) return false;
    if (c.rowptr) {
        int lo, hi;
        group_rows(c.rowptr, c.base, c.S, e, lo, hi);
        if (lo == hi) return false;
    }
    s = (const T *)c.src + e * c.stride;
    if (c.idx) {
        sr = (int64_t)__ldg(c.idx + sr) - c.base;
        if (sr < 0 || sr >= c.limit) {
            outside = true;
            s = nullptr;
            return true;
        }
    }
    s += sr * c.ld;
    return true;
}

// Rows of bf16 to a leading dimension of a multiple of 8: those whose leading
// dimension or address TMA cannot take, and the gradient's gathered rows.  A
// warp moves 1024 neighbouring elements of a row, its loads on the way
// together: 16 bytes a lane where the source is aligned, else 64 bytes a load.
constexpr int kAlignPiece = 1024;
__device__ __forceinline__ void align_piece(const Copy &c, int64_t w, bool &outside) {
    const int lane = threadIdx.x % kWarp;
    int64_t r, p0;
    const uint16_t *s;
    if (!copy_source(c, w, kAlignPiece, r, p0, s, outside)) return;
    uint16_t *d = (uint16_t *)c.dst + r * c.ldd;
    const int n = (int)(c.cols - p0 < kAlignPiece ? c.cols - p0 : kAlignPiece);
    if (c.vec) {
        uint4 v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int k = q * 256 + 8 * lane;
            v[q] = make_uint4(0, 0, 0, 0);
            if (s && k + 8 <= n) v[q] = __ldg(reinterpret_cast<const uint4 *>(s + p0 + k));
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int k = q * 256 + 8 * lane;
            if (k + 8 <= n) *reinterpret_cast<uint4 *>(d + p0 + k) = v[q];
        }
        const int k = (n & ~7) + lane;            // the row's last elements
        if (lane < 8 && k < n) d[p0 + k] = s ? s[p0 + k] : (uint16_t)0;
        return;
    }
#pragma unroll 2
    for (int q0 = 0; q0 < n; q0 += 512) {
        uint16_t v[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) v[q] = s && q0 + q * 32 + lane < n ? s[p0 + q0 + q * 32 + lane] : (uint16_t)0;
#pragma unroll
        for (int q = 0; q < 16; ++q)
            if (q0 + q * 32 + lane < n) d[p0 + q0 + q * 32 + lane] = v[q];
    }
}

// F32 rows as three bf16 planes, h + m + l = the value: h holds its upper 8
// bits, m the next 8 and l the last 8.  Truncated, not rounded, so that h
// cannot overflow and the three have one sign (an overflow stays an infinity).
// An infinity or NaN goes to l, whose only partner is the other operand's h
// (never 0 for a value of 2^-133 or more, +-1 for an infinity), with h = +-1
// for an infinity there; in h it would meet zero m and l planes.
constexpr int kSplitPiece = 512;
__device__ __forceinline__ void split_piece(const Copy &c, int64_t w, bool &outside) {
    const int lane = threadIdx.x % kWarp;
    int64_t r, p0;
    const float *s;
    if (!copy_source(c, w, kSplitPiece, r, p0, s, outside)) return;
    __nv_bfloat16 *dst = (__nv_bfloat16 *)c.dst + r * c.ldd + p0;
    const int64_t plane = c.experts * c.rows * c.ldd;
    const int n = (int)(c.cols - p0 < kSplitPiece ? c.cols - p0 : kSplitPiece);
    float v[2][8];                                // a lane's 8 neighbours, twice
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int k = q * 256 + 8 * lane;
        if (c.vec && s && k + 8 <= n) {
            *reinterpret_cast<float4 *>(v[q]) = __ldg(reinterpret_cast<const float4 *>(s + p0 + k));
            *reinterpret_cast<float4 *>(v[q] + 4) = __ldg(reinterpret_cast<const float4 *>(s + p0 + k + 4));
        } else {
#pragma unroll
            for (int x = 0; x < 8; ++x) v[q][x] = s && k + x < n ? s[p0 + k + x] : 0.0f;
        }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int k = q * 256 + 8 * lane;
        if (k >= n) continue;
        __nv_bfloat162 o[3][4];
#pragma unroll
        for (int x = 0; x < 8; x += 2) {
            float h[2], m[2], l[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const float t = v[q][x + y];
                const uint32_t u = __float_as_uint(t);
                h[y] = __uint_as_float(u & 0xffff0000u);
                const float rest = t - h[y];
                m[y] = __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
                l[y] = rest - m[y];
                if ((u & 0x7f800000u) == 0x7f800000u) {
                    h[y] = copysignf(1.0f, t);
                    m[y] = 0.0f;
                    l[y] = t;
                }
            }
            o[0][x / 2] = __floats2bfloat162_rn(h[0], h[1]);
            o[1][x / 2] = __floats2bfloat162_rn(m[0], m[1]);
            o[2][x / 2] = __floats2bfloat162_rn(l[0], l[1]);
        }
        // whole groups of 8: the copy's rows are padded to them
#pragma unroll
        for (int x = 0; x < 3; ++x) *reinterpret_cast<uint4 *>(dst + x * plane + k) = *reinterpret_cast<const uint4 *>(o[x]);
    }
}

// One or two operands' copies in one launch, their pieces in turn.
template <bool SPLIT>
__global__ void __launch_bounds__(256) copy_rows(const Copy a, const Copy b) {
    bool outside = false;
    const int64_t all = a.warps + b.warps;
    for (int64_t w = (int64_t)blockIdx.x * 8 + threadIdx.x / kWarp; w < all; w += (int64_t)gridDim.x * 8) {
        const bool first = w < a.warps;
        if (SPLIT) split_piece(first ? a : b, first ? w : w - a.warps, outside);
        else align_piece(first ? a : b, first ? w : w - a.warps, outside);
    }
    if (outside) dev_error(DEV_ERR_BOUNDS);
}

static Copy make_copy(bool split, const void *src, int64_t experts, int64_t rows, int64_t cols, int64_t ld,
                      int64_t stride, void *dst) {
    Copy c{};
    c.src = src;
    c.experts = experts;
    c.rows = rows;
    c.cols = cols;
    c.ld = ld;
    c.stride = stride;
    c.vec = tma_rows(src, ld) && (experts == 1 || stride % 8 == 0);
    c.dst = dst;
    c.ldd = pad8(cols);
    c.warps = experts * rows * ceil_div(cols, split ? kSplitPiece : kAlignPiece);
    return c;
}

static int launch_copies(cudaStream_t st, bool split, const Copy &a, const Copy &b) {
    const int64_t blocks = ceil_div(a.warps + b.warps, 8);
    if (blocks == 0) return JLB_OK;
    const unsigned grid = (unsigned)(blocks < 148 * 16 ? blocks : 148 * 16);
    if (split) copy_rows<true><<<grid, 256, 0, st>>>(a, b);
    else copy_rows<false><<<grid, 256, 0, st>>>(a, b);
    JLB_LAUNCH_CHECK("copy_rows");
    return JLB_OK;
}

// The tensor path of a product: which operands need an aligned copy (BF16) or
// are split into planes (F32), and where the workspace holds them (after the
// parts of split tiles).
struct ProductPlan {
    bool tc, split, copy_x, copy_w;
    size_t x_at, w_at, bytes;
    Product p;              // with the copies' leading dimensions
};
static ProductPlan plan_product(const Product &P) {
    ProductPlan q{};
    q.p = P;
    if (P.K == 0 || P.N == 0 || P.S == 0 || P.T == 0 || P.E == 0 || skinny_ok(P)) return q;
    const int64_t inner = P.w_order == JLB_ROW_MAJOR ? P.N : P.K, outer = P.w_order == JLB_ROW_MAJOR ? P.K : P.N;
    q.split = P.dtype == JLB_F32;
    const int64_t planes = q.split ? 3 : 1, xrows = q.split ? P.S : P.T;   // planes of gathered rows
    if (planes * xrows > INT32_MAX / 2 || planes * P.E > INT32_MAX / 2) return q;
    q.tc = true;
    q.copy_x = q.split || !tma_rows(P.x, P.ldx);
    q.copy_w = q.split || !tma_rows(P.w, P.ldw) || (P.E > 1 && P.w_stride % 8);
    q.bytes = pad256(tc_product_workspace(P));
    if (q.copy_x) {
        q.x_at = q.bytes;
        q.bytes += pad256((size_t)(planes * xrows * pad8(P.K)) * 2);
        q.p.ldx = pad8(P.K);
    }
    if (q.copy_w) {
        q.w_at = q.bytes;
        q.bytes += pad256((size_t)(planes * P.E * outer * pad8(inner)) * 2);
        q.p.ldw = pad8(inner);
        q.p.w_stride = outer * pad8(inner);
    }
    return q;
}

static int run_product(cudaStream_t st, const Product &P, void *ws, size_t ws_bytes) {
    if (skinny_ok(P) && P.T > 0) return skinny_product(st, P);
    ProductPlan q = plan_product(P);
    if (q.tc) {
        if (!workspace_ok(ws, ws_bytes, q.bytes))
            return fail(JLB_ERR_WORKSPACE, "the product needs %zu workspace bytes, 16-byte aligned", q.bytes);
        const bool row = P.w_order == JLB_ROW_MAJOR;
        char *base = (char *)ws;
        Copy x{}, w{};
        if (q.copy_x) {
            x = make_copy(q.split, P.x, 1, q.split ? P.S : P.T, P.K, P.ldx, 0, base + q.x_at);
            if (q.split) {                        // planes of the rows already gathered
                x.idx = P.rows;
                x.limit = P.T;
                x.base = P.base;
                x.live_end = P.rowptr ? P.rowptr + P.E : nullptr;
                q.p.rows = nullptr;
                q.p.T = P.S;
            }
        }
        if (q.copy_w) {
            w = make_copy(q.split, P.w, P.E, row ? P.K : P.N, row ? P.N : P.K, P.ldw, P.w_stride, base + q.w_at);
            w.rowptr = P.rowptr;
            w.S = P.S;
            w.base = P.base;
        }
        int r = launch_copies(st, q.split, x, w);
        if (r) return r;
        if (q.copy_x) q.p.x = base + q.x_at;
        if (q.copy_w) q.p.w = base + q.w_at;
        r = tc_product(st, q.p, base);
        if (r >= 0) return r;
    }
    const int64_t ntiles = ceil_div(P.N, kTile), rtiles = row_tiles_bound(P.E, P.S, P.rowptr, kTile);
    const dim3 grid = in_yz(ntiles, rtiles);
    if (P.dtype == JLB_F32) product_simt<float><<<grid, kSimtThreads, 0, st>>>(P);
    else product_simt<__nv_bfloat16><<<grid, kSimtThreads, 0, st>>>(P);
    JLB_LAUNCH_CHECK("product_simt");
    return ok();
}

struct GradientPlan {
    bool tc, split, copy_x, copy_d;
    size_t x_at, d_at, bytes;
    Gradient g;
};
static GradientPlan plan_gradient(const Gradient &G) {
    GradientPlan q{};
    q.g = G;
    if (G.S == 0 || G.T == 0 || G.E == 0 || G.K == 0 || G.N == 0) return q;
    q.split = G.dtype == JLB_F32;
    const int64_t planes = q.split ? 3 : 1, xrows = G.S;
    if (planes * G.S > INT32_MAX / 2) return q;
    q.tc = true;
    // gathered rows are copied too: every tile of the group reads them, by TMA
    // from the copy at 1.3 PFLOP/s, by row loads at 0.85 (8192 x 4096 x 4096)
    q.copy_x = q.split || G.rows || !tma_rows(G.x, G.ldx);
    q.copy_d = q.split || !tma_rows(G.dz, G.lddz);
    q.bytes = pad256(tc_gradient_workspace(G));
    if (q.copy_x) {
        q.x_at = q.bytes;
        q.bytes += pad256((size_t)(planes * xrows * pad8(G.K)) * 2);
        q.g.ldx = pad8(G.K);
    }
    if (q.copy_d) {
        q.d_at = q.bytes;
        q.bytes += pad256((size_t)(planes * G.S * pad8(G.N)) * 2);
        q.g.lddz = pad8(G.N);
    }
    return q;
}

static int run_gradient(cudaStream_t st, const Gradient &G, void *ws, size_t ws_bytes) {
    GradientPlan q = plan_gradient(G);
    if (q.tc) {
        if (!workspace_ok(ws, ws_bytes, q.bytes))
            return fail(JLB_ERR_WORKSPACE, "the gradient needs %zu workspace bytes, 16-byte aligned", q.bytes);
        char *base = (char *)ws;
        Copy x{}, d{};
        if (q.copy_x) {
            x = make_copy(q.split, G.x, 1, G.S, G.K, G.ldx, 0, base + q.x_at);
            x.idx = G.rows;
            x.limit = G.T;
            q.g.rows = nullptr;
            q.g.T = G.S;
        }
        if (q.copy_d) d = make_copy(q.split, G.dz, 1, G.S, G.N, G.lddz, 0, base + q.d_at);
        x.base = d.base = G.base;
        x.live_end = d.live_end = G.rowptr ? G.rowptr + G.E : nullptr;
        int r = launch_copies(st, q.split, x, d);
        if (r) return r;
        if (q.copy_x) q.g.x = base + q.x_at;
        if (q.copy_d) q.g.dz = base + q.d_at;
        r = tc_gradient(st, q.g, base);
        if (r >= 0) return r;
    }
    const bool col = G.w_order == JLB_COL_MAJOR;
    const int64_t mt = ceil_div(col ? G.N : G.K, kTile), nt = ceil_div(col ? G.K : G.N, kTile);
    const dim3 grid((unsigned)nt, (unsigned)(mt < 65535 ? mt : 65535), (unsigned)(G.E < 65535 ? G.E : 65535));
    if (G.dtype == JLB_F32) gradient_simt<float><<<grid, kSimtThreads, 0, st>>>(G);
    else gradient_simt<__nv_bfloat16><<<grid, kSimtThreads, 0, st>>>(G);
    JLB_LAUNCH_CHECK("gradient_simt");
    return ok();
}

// Checks that need every argument of one call.
static int check_call(const Product &P) {
    int r = check_extents(P.E, P.S, P.T, P.K, P.N, P.rowptr, P.rows);
    if (r) return r;
    if (P.ldx < P.K || P.ldy < P.N || (P.z && P.ldz < P.N) || (P.res && P.ldr < P.N))
        return fail(JLB_ERR_INCOMPATIBLE_EXTENTS, "leading dimension too small");
    if (P.S == 0 || P.N == 0) return JLB_OK;
    if (P.E == 0 && P.S > 0)
        return fail(JLB_ERR_INCOMPATIBLE_EXTENTS, "rows without a group (E = 0)");
    if (!P.y || (P.K > 0 && (!P.w || (P.T > 0 && !P.x))))
        return fail(JLB_ERR_INVALID_ARGUMENT, "null buffer");
    return JLB_OK;
}

}  // namespace emm
}  // namespace jlb

using namespace jlb;

struct jlb_mm_plan_s {
    emm::Product p;
};

extern "C" JLB_API int jlb_mm_plan_create(jlb_mm_plan *plan, int dtype, int idx_base, int64_t E,
                                          int64_t K, int64_t N, const void *w, int64_t ldw,
                                          int64_t w_stride, int w_order, const void *bias,
                                          int64_t ldb, int act) {
    if (!plan) return fail(JLB_ERR_INVALID_ARGUMENT, "null plan");
    *plan = nullptr;
    int r = emm::check_types(dtype, idx_base);
    if (!r) r = emm::check_act(act);
    if (!r && (E < 0 || K < 0 || N < 0)) r = fail(JLB_ERR_INCOMPATIBLE_EXTENTS, "negative extent");
    if (!r) r = emm::check_weight(w_order, E, K, N, ldw, w_stride);
    if (!r && bias && E > 1 && ldb < N)
        r = fail(JLB_ERR_INCOMPATIBLE_EXTENTS, "bias leading dimension too small");
    if (!r && E * K * N > 0 && !w) r = fail(JLB_ERR_INVALID_ARGUMENT, "null weights");
    if (r) return r;
    jlb_mm_plan_s *h = new (std::nothrow) jlb_mm_plan_s();
    if (!h) return fail(JLB_ERR_CUDA, "out of host memory");
    emm::Product &p = h->p;
    p = emm::Product{};
    p.dtype = dtype;
    p.base = idx_base;
    p.act = act;
    p.w_order = w_order;
    p.E = E;
    p.K = K;
    p.N = N;
    p.w = w;
    p.ldw = ldw;
    p.w_stride = w_stride;
    p.bias = bias;
    p.ldb = ldb;
    *plan = h;
    return ok();
}

extern "C" JLB_API int jlb_mm_plan_destroy(jlb_mm_plan plan) {
    delete plan;
    return ok();
}

extern "C" JLB_API size_t jlb_mm_plan_workspace_size(jlb_mm_plan plan, int64_t S, int64_t T,
                                                     const void *x, int64_t ldx, int gather) {
    if (!plan || S < 0 || T < 0) return 0;
    emm::Product P = plan->p;
    P.S = S;
    P.T = T;
    P.x = x;
    P.ldx = ldx;
    (void)gather;
    // with and without a row pointer, which is not known here: the larger
    static const int32_t some = 0;
    const size_t dense = P.E == 1 ? emm::plan_product(P).bytes : 0;
    P.rowptr = &some;
    const size_t ragged = emm::plan_product(P).bytes;
    return dense > ragged ? dense : ragged;
}

extern "C" JLB_API int jlb_mm_plan_execute(jlb_mm_plan plan, void *stream, int64_t S, int64_t T,
                                           const int32_t *rowptr, const int32_t *rows,
                                           const void *x, int64_t ldx, const void *res,
                                           int64_t ldr, void *z, int64_t ldz, void *y, int64_t ldy,
                                           void *workspace, size_t workspace_bytes) {
    if (!plan) return fail(JLB_ERR_INVALID_ARGUMENT, "null plan");
    emm::Product P = plan->p;
    P.S = S;
    P.T = T;
    P.rowptr = rowptr;
    P.rows = rows;
    P.x = x;
    P.ldx = ldx;
    P.res = res;
    P.ldr = ldr;
    P.z = z;
    P.ldz = ldz;
    P.y = y;
    P.ldy = ldy;
    const int r = emm::check_call(P);
    if (r) return r;
    if (S == 0 || P.N == 0) return ok();
    return emm::run_product(as_stream(stream), P, workspace, workspace_bytes);
}

extern "C" JLB_API size_t jlb_grouped_mm_workspace_size(int dtype, int64_t E, int64_t S, int64_t T,
                                                        int64_t K, int64_t N, const void *x,
                                                        int64_t ldx, const void *w, int64_t ldw,
                                                        int64_t w_stride, int w_order, int gather) {
    if (E < 0 || K < 0 || N < 0) return 0;
    jlb_mm_plan_s h;
    h.p = emm::Product{};
    h.p.dtype = dtype;
    h.p.E = E;
    h.p.K = K;
    h.p.N = N;
    h.p.w = w;
    h.p.ldw = ldw;
    h.p.w_stride = w_stride;
    h.p.w_order = w_order;
    return jlb_mm_plan_workspace_size(&h, S, T, x, ldx, gather);
}

extern "C" JLB_API int jlb_grouped_mm(void *stream, int dtype, int idx_base, int64_t E, int64_t S,
                                      int64_t T, int64_t K, int64_t N, const int32_t *rowptr,
                                      const int32_t *rows, const void *x, int64_t ldx,
                                      const void *w, int64_t ldw, int64_t w_stride, int w_order,
                                      const void *bias, int64_t ldb, int act, const void *res,
                                      int64_t ldr, void *z, int64_t ldz, void *y, int64_t ldy,
                                      void *workspace, size_t workspace_bytes) {
    jlb_mm_plan h = nullptr;
    int r = jlb_mm_plan_create(&h, dtype, idx_base, E, K, N, w, ldw, w_stride, w_order, bias, ldb, act);
    if (r) return r;
    r = jlb_mm_plan_execute(h, stream, S, T, rowptr, rows, x, ldx, res, ldr, z, ldz, y, ldy,
                            workspace, workspace_bytes);
    delete h;
    return r;
}

extern "C" JLB_API size_t jlb_grouped_mm_wgrad_workspace_size(int dtype, int64_t E, int64_t S,
                                                              int64_t T, int64_t K, int64_t N,
                                                              const void *x, int64_t ldx,
                                                              const void *dz, int64_t lddz,
                                                              int w_order, int gather) {
    static const int32_t some = 0;
    if (E < 0 || S < 0 || T < 0 || K < 0 || N < 0) return 0;
    emm::Gradient G{};
    G.dtype = dtype;
    G.E = E;
    G.S = S;
    G.T = T;
    G.K = K;
    G.N = N;
    G.x = x;
    G.ldx = ldx;
    G.dz = dz;
    G.lddz = lddz;
    G.w_order = w_order;
    G.rows = gather ? &some : nullptr;
    return emm::plan_gradient(G).bytes;
}

extern "C" JLB_API int jlb_grouped_mm_wgrad(void *stream, int dtype, int idx_base, int64_t E,
                                            int64_t S, int64_t T, int64_t K, int64_t N,
                                            const int32_t *rowptr, const int32_t *rows,
                                            const void *x, int64_t ldx, const void *dz,
                                            int64_t lddz, void *dw, int64_t lddw,
                                            int64_t dw_stride, int w_order, void *workspace,
                                            size_t workspace_bytes) {
    int r = emm::check_types(dtype, idx_base);
    if (!r) r = emm::check_extents(E, S, T, K, N, rowptr, rows);
    if (!r) r = emm::check_weight(w_order, E, K, N, lddw, dw_stride);
    if (!r && (ldx < K || lddz < N))
        r = fail(JLB_ERR_INCOMPATIBLE_EXTENTS, "leading dimension too small");
    if (r) return r;
    if (E == 0 || K == 0 || N == 0) return ok();
    if (!dw || (S > 0 && (!dz || (T > 0 && !x)))) return fail(JLB_ERR_INVALID_ARGUMENT, "null buffer");
    const emm::Gradient G{dtype, idx_base, w_order, E, S, T, K, N, rowptr, rows,
                          x, ldx, dz, lddz, dw, lddw, dw_stride};
    return emm::run_gradient(as_stream(stream), G, workspace, workspace_bytes);
}

extern "C" JLB_API size_t jlb_act_backward_workspace_size(int64_t E, int64_t S, int64_t N,
                                                          int need_db) {
    if (!need_db || E <= 0 || S <= 0 || N <= 0) return 0;
    return (size_t)(emm::row_tiles_bound(E, S, true, emm::kSumRows) * N * 4);
}

extern "C" JLB_API int jlb_act_backward(void *stream, int dtype, int idx_base, int64_t E, int64_t S,
                                        int64_t N, const int32_t *rowptr, int act, const void *dy,
                                        int64_t lddy, const void *z, int64_t ldz, void *dz,
                                        int64_t lddz, void *db, int64_t lddb, void *workspace,
                                        size_t workspace_bytes) {
    int r = emm::check_types(dtype, idx_base);
    if (!r) r = emm::check_act(act);
    if (!r) r = emm::check_extents(E, S, S, 0, N, rowptr, nullptr);
    if (r) return r;
    if (lddy < N || (z && ldz < N) || (dz && lddz < N) || (db && E > 1 && lddb < N))
        return fail(JLB_ERR_INCOMPATIBLE_EXTENTS, "leading dimension too small");
    if (act != JLB_ACT_NONE && !z && S > 0 && N > 0)
        return fail(JLB_ERR_INVALID_ARGUMENT, "an activation's gradient needs the pre-activation");
    if (N == 0 || E == 0 || (!dz && !db)) return ok();
    if (S > 0 && !dy) return fail(JLB_ERR_INVALID_ARGUMENT, "null buffer");
    const size_t need = jlb_act_backward_workspace_size(E, S, N, db != nullptr);
    if (!workspace_ok(workspace, workspace_bytes, need))
        return fail(JLB_ERR_WORKSPACE, "act_backward needs %zu workspace bytes, 16-byte aligned", need);
    if (act == JLB_ACT_NONE) z = nullptr;
    cudaStream_t st = as_stream(stream);
    const int64_t tiles = emm::row_tiles_bound(E, S, rowptr, emm::kSumRows);
    float *part = db ? (float *)workspace : nullptr;
    if (tiles > 0) {
        r = dtype == JLB_F32 ? emm::launch_act<float>(st, tiles, E, S, N, idx_base, rowptr, act, dy, lddy, z, ldz, dz, lddz, part)
                             : emm::launch_act<__nv_bfloat16>(st, tiles, E, S, N, idx_base, rowptr, act, dy, lddy, z, ldz,
                                                              dz, lddz, part);
        if (r) return r;
    }
    if (db) {
        const dim3 grid = emm::in_yz(ceil_div(N, 256), E);
        if (dtype == JLB_F32)
            emm::sum_parts<float><<<grid, 256, 0, st>>>(E, S, N, idx_base, rowptr, part, tiles,
                                                        (float *)db, lddb);
        else
            emm::sum_parts<__nv_bfloat16><<<grid, 256, 0, st>>>(E, S, N, idx_base, rowptr, part, tiles,
                                                                (__nv_bfloat16 *)db, lddb);
        JLB_LAUNCH_CHECK("sum_parts");
    }
    return ok();
}
