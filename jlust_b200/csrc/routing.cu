// routing.cu -- the routing pattern of a layer of experts and the products
// with it.  A token's k expert indices are one row of a sparse T x E matrix R;
// its pattern compressed by column (expert) gives each expert's rows, and
// slot[t, j] is where entry (t, j) landed in that order.
#include "common.cuh"

namespace jlb {

JLB_DEFINE_DEV_ERROR(routing)

namespace routing {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / kWarp;
constexpr int kPer = 4;                       // entries a thread
constexpr int kChunk = kThreads * kPer;       // entries a CTA
constexpr int kMaxE = 2048;
// Whether the chunks' counts are scanned by kernels of their own (three launches
// more) instead of being added up by every CTA: each adds chunks x E counts, in as
// many rounds as the SMs, one CTA each, need for the chunks.  A call among other
// work, caches cold, added up against scanned: one round, 64 x 256 17 against
// 28 us, 118 x 256 24 against 28, 128 x 512 32 against 30, 64 x 1,024 32 against
// 34, 128 x 1,024 48 against 34, 32 x 2,048 38 against 42, 64 x 2,048 52 against
// 42; two, 192 x 128 34 against 34, 256 x 64 30 against 34, 256 x 128 38 against
// 34, 160 x 256 42 against 36; three and four, 384 x 64 46 against 44, 512 x 16
// 42 against 46, 512 x 64 65 against 48, 512 x 2,048 861 against 112.
__host__ __device__ constexpr bool scans_counts(int64_t chunks, int64_t E) {
    return (chunks + 147) / 148 * chunks * E >= 65536;
}

// The expert of entry i, or -1 when it is dropped (outside 0 .. E-1).
__device__ __forceinline__ int expert_of(const int32_t *__restrict__ ids, int64_t i, int64_t n,
                                         int base, int E) {
    if (i >= n) return -1;
    const int e = __ldg(ids + i) - base;
    return e >= 0 && e < E ? e : -1;
}

// Entry order inside a CTA's chunk: warp w holds entries w*128 .. w*128+127,
// lane l of round r entry w*128 + r*32 + l, so (warp, round, lane) ascends
// with the entry index.
__device__ __forceinline__ int64_t entry_index(int warp, int round, int lane) {
    return (int64_t)blockIdx.x * kChunk + warp * (kWarp * kPer) + round * kWarp + lane;
}

// Entries per expert of each chunk: hist[chunk * cs + e * es].
__global__ void __launch_bounds__(kThreads) route_count(const int32_t *__restrict__ ids, int64_t n,
                                                        int base, int E, int64_t cs, int64_t es,
                                                        int32_t *__restrict__ hist) {
    extern __shared__ int32_t cnt[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int e = threadIdx.x; e < E; e += kThreads) cnt[e] = 0;
    __syncthreads();
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
        const int e = expert_of(ids, entry_index(warp, r, lane), n, base, E);
        if (e >= 0) atomicAdd(&cnt[e], 1);    // a sum of ones: the same in any order
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kThreads) hist[blockIdx.x * cs + e * es] = cnt[e];
}

// Places the entries.  Stable counting sort by expert: slot(i) = entries of
// smaller experts + entries of the same expert in earlier chunks, earlier
// warps of the chunk and earlier entries of the warp.  With one chunk
// (hist == nullptr) the counts come from the warps' own; with several
// every CTA adds up the chunks' counts itself, or `at` holds their scan, expert
// by expert (E x chunks; scans_counts).
__global__ void __launch_bounds__(kThreads)
route_place(const int32_t *__restrict__ ids, int64_t n, int k, int base, int E,
            const int32_t *hist, const int32_t *__restrict__ at, int chunks,
            int32_t *__restrict__ rowptr, int32_t *__restrict__ source, int32_t *__restrict__ slot) {
    extern __shared__ int32_t sm[];
    int32_t *tot = sm;                        // E: entries per expert, then their exclusive scan
    int32_t *mine = tot + E;                  // E: entries of earlier chunks
    uint16_t *wh = reinterpret_cast<uint16_t *>(mine + E);   // kWarps x E: the warps' counts
    __shared__ int32_t wsum[kWarps];
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    for (int i = threadIdx.x; i < kWarps * E / 2; i += kThreads) reinterpret_cast<uint32_t *>(wh)[i] = 0;
    __syncthreads();
    // ranks inside the warp, in entry order (a dropped entry is expert -1: all
    // bits set, which no expert below 2^bits - 1 has)
    const int bits = 32 - __clz(E);
    int ex[kPer], rank[kPer];
    uint16_t *my = wh + warp * E;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
        ex[r] = expert_of(ids, entry_index(warp, r, lane), n, base, E);
        // lanes of the same expert, a ballot a bit (match.any takes a step for
        // each distinct value, up to 32 here)
        unsigned same = 0xffffffffu;
        for (int b = 0; b < bits; ++b) {
            const unsigned set = __ballot_sync(0xffffffffu, ex[r] >> b & 1);
            same &= ex[r] >> b & 1 ? set : ~set;
        }
        const int before = __popc(same & ((1u << lane) - 1u));
        int have = 0;
        if (ex[r] >= 0) have = my[ex[r]];
        __syncwarp();
        if (ex[r] >= 0 && before == 0) my[ex[r]] = (uint16_t)(have + __popc(same));
        __syncwarp();
        rank[r] = have + before;
    }
    __syncthreads();
    // counts over the warps become each warp's offset inside the chunk; with
    // several chunks, kThreads / E threads an expert add up the chunks' counts
    // (four neighbouring threads an expert, eight warps each)
    for (int i = threadIdx.x; i < 4 * E; i += kThreads) {
        const int e = i / 4, w0 = (i & 3) * (kWarps / 4);
        int c[kWarps / 4], sum = 0;
#pragma unroll
        for (int w = 0; w < kWarps / 4; ++w) sum += c[w] = wh[(w0 + w) * E + e];
        const unsigned peers = 0xfu << (lane & ~3);
        int run = 0, all = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int s = __shfl_sync(peers, sum, (lane & ~3) + q);
            if (q < (i & 3)) run += s;
            all += s;
        }
#pragma unroll
        for (int w = 0; w < kWarps / 4; ++w) {
            wh[(w0 + w) * E + e] = (uint16_t)run;
            run += c[w];
        }
        if ((i & 3) == 0) {
            tot[e] = hist || at ? 0 : all;
            mine[e] = 0;
        }
    }
    __syncthreads();
    if (hist) {
        asm volatile("griddepcontrol.wait;" ::: "memory");      // the chunks' counts are complete
        const int per = E < kThreads ? kThreads / E : 1;
        for (int i = threadIdx.x; i < per * E; i += kThreads) {
            const int e = i % E, p = i / E;
            int all = 0, before = 0;
#pragma unroll 8
            for (int c = p; c < chunks; c += per) {
                // coherent: route_count writes them while this grid runs
                const int h = __ldcg(hist + (int64_t)c * E + e);
                if (c < (int)blockIdx.x) before += h;
                all += h;
            }
            atomicAdd(&tot[e], all);              // integers: the same in any order
            atomicAdd(&mine[e], before);
        }
        __syncthreads();
    }
    int carry = 0;
    if (at) {
        for (int e = threadIdx.x; e < E; e += kThreads) {
            tot[e] = __ldg(at + (int64_t)e * chunks);
            mine[e] = __ldg(at + (int64_t)e * chunks + blockIdx.x) - tot[e];
            if (blockIdx.x == 0) rowptr[e] = tot[e] + base;
        }
        carry = __ldg(at + (int64_t)E * chunks);
        __syncthreads();
    }
    // exclusive scan of tot over the experts, kThreads at a time
    for (int e0 = 0; !at && e0 < E; e0 += kThreads) {
        const int e = e0 + threadIdx.x;
        const int v = e < E ? tot[e] : 0;
        int inc = v;
#pragma unroll
        for (int o = 1; o < kWarp; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        if (lane == kWarp - 1) wsum[warp] = inc;
        __syncthreads();
        if (warp == 0) {
            int s = wsum[lane];
#pragma unroll
            for (int o = 1; o < kWarp; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += u;
            }
            wsum[lane] = s;
        }
        __syncthreads();
        const int excl = carry + (warp ? wsum[warp - 1] : 0) + inc - v;
        if (e < E) {
            tot[e] = excl;
            if (blockIdx.x == 0) rowptr[e] = excl + base;
        }
        carry += wsum[kWarps - 1];
        __syncthreads();
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) rowptr[E] = carry + base;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
        const int64_t i = entry_index(warp, r, lane);
        if (i >= n) continue;
        const int e = ex[r];
        if (e >= 0) {
            const int p = tot[e] + mine[e] + my[e] + rank[r];
            slot[i] = p + base;
            source[p] = (int32_t)(i / k) + base;
        } else {
            slot[i] = base - 1;
        }
        if (i >= carry) source[i] = base - 1;    // slots that no entry took
    }
}

// ------------------------------------------------------------ value access
// V neighbouring values (16 bytes, or one) as they lie in memory, so that
// several rows' loads can wait in few registers.
template <typename T, int V>
struct Raw {
    uint4 q;
    T one;
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (V == 1) one = *p;
        else q = __ldg(reinterpret_cast<const uint4 *>(p));
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (V == 1) {
            if constexpr (sizeof(T) == 2) return __bfloat162float(one);
            else return one;
        } else {
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
            if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
            else return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        }
    }
};
template <typename T, int V>
__device__ __forceinline__ void store_values(T *p, const float (&v)[V]) {
    if constexpr (V == 1) {
        if constexpr (sizeof(T) == 2) *p = __float2bfloat16_rn(v[0]);
        else *p = v[0];
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// y[t] = sum_j g[t, j] z[slot[t, j]] in the order of j, fp32 sums rounded
// once to the value type.  V columns a thread (16 bytes, or one when the
// layout is not aligned); blockDim = (column threads, tokens).
constexpr int kCombineThreads = 128;
// R rows of C column groups are under way in a thread.  Bound by HBM: 8191
// tokens x 4 rows of 4096 bf16 55 us (floor 52; 58 with R = 4, C = 2 and CTAs
// of 256), 16,384 x 2 of 2048 36 us (floor 31; 46 with R = 4, C = 2), 8192 x 3
// of 2048 24 us with R = 3 (27 with R = 2).  A value a load is bound by the
// loads' number: 16,384 x 4 rows of 1001 bf16 59 us (floor 25; 71 with C = 4);
// 16-byte blocks shifted into place took 52 us there and more elsewhere.
template <typename T, int V, int R, int C>
__global__ void __launch_bounds__(kCombineThreads)
combine_rows(int64_t T_, int k, int64_t S, int64_t N, int base, const int32_t *__restrict__ slot,
             const float *__restrict__ g, const T *__restrict__ z, int64_t ldz,
             T *__restrict__ y, int64_t ldy) {
    const int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (t >= T_) return;
    const int32_t *sl = slot + t * k;
    const int64_t step = (int64_t)blockDim.x * V;       // from one of a thread's column groups to the next
    for (int64_t c = (int64_t)blockIdx.y * step * C + threadIdx.x * V; c < N; c += (int64_t)gridDim.y * step * C) {
        float acc[C][V];
#pragma unroll
        for (int x = 0; x < C; ++x)
#pragma unroll
            for (int i = 0; i < V; ++i) acc[x][i] = 0.0f;
        for (int j0 = 0; j0 < k; j0 += R) {      // their loads on the way together
            Raw<T, V> v[R][C];
            float w[R];
            int p[R];                                     // slots, -1: none
            // all slots before any row, so that no row waits for the next slot
#pragma unroll
            for (int q = 0; q < R; ++q) {
                p[q] = -1;
                w[q] = 0.0f;
                if (j0 + q < k) {
                    const int64_t at = (int64_t)__ldg(sl + j0 + q) - base;
                    w[q] = g ? __ldg(g + t * k + j0 + q) : 1.0f;
                    if (at >= S) dev_error(DEV_ERR_BOUNDS);
                    p[q] = at < 0 || at >= S ? -1 : (int)at;      // a dropped entry has no slot
                }
            }
#pragma unroll
            for (int x = 0; x < C; ++x)
                if (c + x * step < N)
#pragma unroll
                    for (int q = 0; q < R; ++q)
                        if (p[q] >= 0) v[q][x].load(z + (int64_t)p[q] * ldz + c + x * step);
#pragma unroll
            for (int q = 0; q < R; ++q)
                if (p[q] >= 0)
#pragma unroll
                    for (int x = 0; x < C; ++x)
#pragma unroll
                        for (int i = 0; i < V; ++i) acc[x][i] = fmaf(w[q], v[q][x].get(i), acc[x][i]);
        }
#pragma unroll
        for (int x = 0; x < C; ++x)
            if (c + x * step < N) store_values<T, V>(y + t * ldy + c + x * step, acc[x]);
    }
}

constexpr int kBwdThreads = 128;

// Rows first, first + step, ... past the last slot.
template <typename T>
__device__ __forceinline__ void clear_rows(int64_t first, int64_t step,
                                           const int32_t *__restrict__ live_end, int base, int64_t S,
                                           int64_t N, T *__restrict__ dz, int64_t lddz) {
    int64_t end = (int64_t)__ldg(live_end) - base;
    end = end < 0 ? 0 : end > S ? S : end;
    for (int64_t p = end + first; p < S; p += step)
        for (int64_t c = (int64_t)threadIdx.x; c < N; c += kBwdThreads) dz[p * lddz + c] = T(0.0f);
}

// dg[j] = the CTA's sum of dot[j] for j < left, by a fixed tree.
template <int J>
__device__ __forceinline__ void write_dots(const float (&dot)[J], int left, float *__restrict__ dg,
                                           float (&part)[kBwdThreads / kWarp][J]) {
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const float s = warp_sum(dot[j]);
        if (lane == 0) part[warp][j] = s;
    }
    __syncthreads();
    if (threadIdx.x < J && (int)threadIdx.x < left) {
        float s = 0.0f;
        for (int q = 0; q < kBwdThreads / kWarp; ++q) s += part[q][threadIdx.x];
        dg[threadIdx.x] = s;
    }
}

// dz[slot[t, j]] = g[t, j] dy[t] and dg[t, j] = <dy[t], z[slot[t, j]]>: one
// CTA a token, dy read once for J entries.  Rows of dz past the last
// slot are zeroed.  The dot product's terms are summed per thread, then by a
// fixed tree over the CTA.
// J follows k, so that registers are left for C column groups under way:
// 16,384 tokens x 2 rows of 2048 bf16 53 us (floor 52) against 83 with J = 8,
// 8191 x 4 of 4096 92 against 101.
template <typename T, int V, int J, int C>
__global__ void __launch_bounds__(kBwdThreads)
combine_bwd(int64_t T_, int k, int64_t S, int64_t N, int base, const int32_t *__restrict__ slot,
            const int32_t *__restrict__ live_end, const float *__restrict__ g,
            const T *__restrict__ z, int64_t ldz, const T *__restrict__ dy, int64_t lddy,
            T *__restrict__ dz, int64_t lddz, float *__restrict__ dg) {
    __shared__ float part[kBwdThreads / kWarp][J];
    const int64_t t = blockIdx.x;
    if (t >= T_) {                                // the CTAs after the tokens: rows of no slot
        clear_rows(t - T_, gridDim.x - T_, live_end, base, S, N, dz, lddz);
        return;
    }
    for (int j0 = 0; j0 < k; j0 += J) {
        int p[J];                              // slots, -1: none
        float w[J], dot[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            p[j] = -1;
            w[j] = dot[j] = 0.0f;
            if (j0 + j < k) {
                const int64_t s = (int64_t)__ldg(slot + t * k + j0 + j) - base;
                w[j] = g ? __ldg(g + t * k + j0 + j) : 1.0f;
                if (s >= S) dev_error(DEV_ERR_BOUNDS);
                p[j] = s < 0 || s >= S ? -1 : (int)s;
            }
        }
        for (int64_t c0 = (int64_t)threadIdx.x * V; c0 < N; c0 += kBwdThreads * V * C) {
            Raw<T, V> d[C], v[J][C];
#pragma unroll
            for (int x = 0; x < C; ++x) {
                const int64_t c = c0 + x * kBwdThreads * V;
                if (c >= N) continue;
                d[x].load(dy + t * lddy + c);
#pragma unroll
                for (int j = 0; j < J; ++j)
                    if (p[j] >= 0) v[j][x].load(z + (int64_t)p[j] * ldz + c);
            }
#pragma unroll
            for (int x = 0; x < C; ++x) {
                const int64_t c = c0 + x * kBwdThreads * V;
                if (c >= N) continue;
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    if (p[j] < 0) continue;
                    float o[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        dot[j] = fmaf(d[x].get(i), v[j][x].get(i), dot[j]);
                        o[i] = w[j] * d[x].get(i);
                    }
                    store_values<T, V>(dz + (int64_t)p[j] * lddz + c, o);
                }
            }
        }
        if (dg) write_dots<J>(dot, k - j0, dg + t * k + j0, part);
    }
}

static size_t place_smem(int64_t E) { return (size_t)E * (8 + 2 * kWarps); }

}  // namespace routing
}  // namespace jlb

using namespace jlb;

extern "C" JLB_API size_t jlb_route_workspace_size(int64_t T, int64_t k, int64_t E) {
    if (T <= 0 || k <= 0 || E <= 0) return 0;
    const int64_t chunks = ceil_div(T * k, routing::kChunk);
    if (chunks <= 1) return 0;
    // many chunks: their counts, the counts' scan and its workspace
    return !routing::scans_counts(chunks, E) ? (size_t)(chunks * E * 4)
                                             : (size_t)(2 * chunks * E + 64) * 4 + conv::scan_ws(chunks * E) + 256;
}

extern "C" JLB_API int jlb_route(void *stream, int idx_base, int64_t T, int64_t k, int64_t E,
                                 const int32_t *ids, int32_t *rowptr, int32_t *source,
                                 int32_t *slot, void *workspace, size_t workspace_bytes) {
    using namespace routing;
    if (idx_base != 0 && idx_base != 1) return fail(JLB_ERR_INVALID_ARGUMENT, "idx_base must be 0 or 1");
    if (T < 0 || k < 0 || E < 0) return fail(JLB_ERR_INCOMPATIBLE_EXTENTS, "negative extent");
    if (E > kMaxE)
        return fail(JLB_ERR_UNSUPPORTED_FORMAT, "more than %d experts (%lld)", kMaxE, (long long)E);
    if (k > 0 && T > (int64_t)(INT32_MAX - kChunk) / k)
        return fail(JLB_ERR_UNSUPPORTED_INDEX_TYPE, "T * k exceeds Int32 positions");
    const int64_t n = T * k;
    if (!rowptr || (n > 0 && (!ids || !source || !slot)))
        return fail(JLB_ERR_INVALID_ARGUMENT, "null buffer");
    const int chunks = (int)ceil_div(n > 0 ? n : 1, kChunk);
    const size_t need = jlb_route_workspace_size(T, k, E);
    if (!workspace_ok(workspace, workspace_bytes, need))
        return fail(JLB_ERR_WORKSPACE, "route needs %zu workspace bytes, 16-byte aligned", need);
    cudaStream_t st = as_stream(stream);
    int32_t *hist = need ? (int32_t *)workspace : nullptr, *at = nullptr;
    if (hist) {
        const bool wide = scans_counts(chunks, E);
        route_count<<<chunks, kThreads, (size_t)E * 4, st>>>(ids, n, idx_base, (int)E, wide ? 1 : E,
                                                             wide ? chunks : 1, hist);
        JLB_LAUNCH_CHECK("route_count");
        if (wide) {
            const int64_t counts = chunks * E;
            at = hist + counts;
            char *ws = (char *)(((uintptr_t)(at + counts + 1) + 255) & ~(uintptr_t)255);
            const int r = conv::scan(st, counts, hist, at, 0, ws, conv::scan_ws(counts));
            if (r) return r;
            hist = nullptr;
        }
    }
    const size_t smem = place_smem(E);
    if (smem > 48 * 1024)
        JLB_CUDA(cudaFuncSetAttribute(route_place, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)smem));
    // starts while the counts are being made and waits for them after its own
    // ranks; alone it is an ordinary launch
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)chunks);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = hist ? 1 : 0;
    JLB_CUDA(cudaLaunchKernelEx(&cfg, route_place, ids, n, (int)(k > 0 ? k : 1), idx_base, (int)E,
                                (const int32_t *)hist, (const int32_t *)at, chunks, rowptr, source, slot));
    return ok();
}

namespace {

int check_combine(int dtype, int idx_base, int64_t T, int64_t k, int64_t S, int64_t N) {
    if (dtype != JLB_F32 && dtype != JLB_BF16)
        return fail(JLB_ERR_UNSUPPORTED_VALUE_TYPE, "combine runs on F32 and BF16 values");
    if (idx_base != 0 && idx_base != 1) return fail(JLB_ERR_INVALID_ARGUMENT, "idx_base must be 0 or 1");
    if (T < 0 || k < 0 || S < 0 || N < 0) return fail(JLB_ERR_INCOMPATIBLE_EXTENTS, "negative extent");
    if (T > INT32_MAX / 2 || S > INT32_MAX || k > INT32_MAX)
        return fail(JLB_ERR_UNSUPPORTED_INDEX_TYPE, "extent exceeds Int32 positions");
    return JLB_OK;
}

template <typename T>
int run_combine(cudaStream_t st, int64_t Tn, int64_t k, int64_t S, int64_t N, int base,
                const int32_t *slot, const float *g, const T *z, int64_t ldz, T *y, int64_t ldy) {
    constexpr int V = 16 / (int)sizeof(T);
    const bool vec = N % V == 0 && ldz % V == 0 && ldy % V == 0 && aligned16(z) && aligned16(y);
    const bool two = k == 2 || k == 4;
    const int64_t items = ceil_div(vec ? N / V : N, !vec ? 8 : k == 1 || two ? 4 : 2);
    int tx = 32;
    while (tx < routing::kCombineThreads && tx < items) tx *= 2;
    const int ty = routing::kCombineThreads / tx;
    const dim3 block(tx, ty);
    const dim3 grid((unsigned)ceil_div(Tn, ty),
                    (unsigned)(ceil_div(items, tx) < 65535 ? ceil_div(items, tx) : 65535));
    // few rows leave registers for more columns; three rows at a time suit the
    // other counts (a fourth would be idle in the last pass)
    const auto kernel = vec ? (k == 1 ? routing::combine_rows<T, V, 1, 4>
                               : two  ? routing::combine_rows<T, V, 2, 4>
                                      : routing::combine_rows<T, V, 3, 2>)
                            : (k == 1 ? routing::combine_rows<T, 1, 1, 8>
                                      : routing::combine_rows<T, 1, 2, 8>);
    kernel<<<grid, block, 0, st>>>(Tn, (int)k, S, N, base, slot, g, z, ldz, y, ldy);
    JLB_LAUNCH_CHECK("combine_rows");
    return ok();
}

template <typename T>
int run_combine_bwd(cudaStream_t st, int64_t Tn, int64_t k, int64_t S, int64_t N, int base,
                    const int32_t *slot, const int32_t *live_end, const float *g, const T *z,
                    int64_t ldz, const T *dy, int64_t lddy, T *dz, int64_t lddz, float *dg) {
    constexpr int V = 16 / (int)sizeof(T);
    const bool vec = N % V == 0 && ldz % V == 0 && lddy % V == 0 && lddz % V == 0 &&
                     aligned16(z) && aligned16(dy) && aligned16(dz);
    const unsigned grid = (unsigned)(Tn + 148);   // 148 CTAs for the rows of no slot
    const auto kernel =
        vec ? (k == 1   ? routing::combine_bwd<T, V, 1, 2>
               : k == 2 ? routing::combine_bwd<T, V, 2, 2>
               : k <= 4 ? routing::combine_bwd<T, V, 4, 2>
                        : routing::combine_bwd<T, V, 8, 1>)
            : (k <= 2   ? routing::combine_bwd<T, 1, 2, 4>
               : k <= 4 ? routing::combine_bwd<T, 1, 4, 4>
                        : routing::combine_bwd<T, 1, 8, 4>);
    kernel<<<grid, routing::kBwdThreads, 0, st>>>(Tn, (int)k, S, N, base, slot, live_end, g, z, ldz,
                                                  dy, lddy, dz, lddz, dg);
    JLB_LAUNCH_CHECK("combine_bwd");
    return ok();
}

}  // namespace

extern "C" JLB_API int jlb_combine(void *stream, int dtype, int idx_base, int64_t T, int64_t k,
                                   int64_t S, int64_t N, const int32_t *slot, const float *g,
                                   const void *z, int64_t ldz, void *y, int64_t ldy) {
    const int r = check_combine(dtype, idx_base, T, k, S, N);
    if (r) return r;
    if (ldz < N || ldy < N) return fail(JLB_ERR_INCOMPATIBLE_EXTENTS, "leading dimension smaller than N");
    if (T == 0 || N == 0) return ok();
    if (!y || (k > 0 && !slot) || (k > 0 && S > 0 && !z))
        return fail(JLB_ERR_INVALID_ARGUMENT, "null buffer");
    cudaStream_t st = as_stream(stream);
    return dtype == JLB_F32 ? run_combine<float>(st, T, k, S, N, idx_base, slot, g, (const float *)z,
                                                 ldz, (float *)y, ldy)
                            : run_combine<__nv_bfloat16>(st, T, k, S, N, idx_base, slot, g,
                                                         (const __nv_bfloat16 *)z, ldz,
                                                         (__nv_bfloat16 *)y, ldy);
}

extern "C" JLB_API int jlb_combine_backward(void *stream, int dtype, int idx_base, int64_t T,
                                            int64_t k, int64_t S, int64_t N, int64_t E,
                                            const int32_t *rowptr, const int32_t *slot,
                                            const float *g, const void *z, int64_t ldz,
                                            const void *dy, int64_t lddy, void *dz, int64_t lddz,
                                            float *dg) {
    const int r = check_combine(dtype, idx_base, T, k, S, N);
    if (r) return r;
    if (E < 0) return fail(JLB_ERR_INCOMPATIBLE_EXTENTS, "negative extent");
    if (ldz < N || lddy < N || lddz < N)
        return fail(JLB_ERR_INCOMPATIBLE_EXTENTS, "leading dimension smaller than N");
    if (S == 0 && T * k == 0) return ok();
    if (!rowptr || (T * k > 0 && (!slot || (N > 0 && !dy) || (S > 0 && N > 0 && !z))) ||
        (S > 0 && N > 0 && !dz))
        return fail(JLB_ERR_INVALID_ARGUMENT, "null buffer");
    cudaStream_t st = as_stream(stream);
    return dtype == JLB_F32
               ? run_combine_bwd<float>(st, T, k, S, N, idx_base, slot, rowptr + E, g,
                                        (const float *)z, ldz, (const float *)dy, lddy, (float *)dz,
                                        lddz, dg)
               : run_combine_bwd<__nv_bfloat16>(st, T, k, S, N, idx_base, slot, rowptr + E, g,
                                                (const __nv_bfloat16 *)z, ldz,
                                                (const __nv_bfloat16 *)dy, lddy,
                                                (__nv_bfloat16 *)dz, lddz, dg);
}
