// paged_select.cu — which blocks of a long context a query should attend (b200_paged_select).
//
// A block's key bounds give an upper bound of q.k over its keys: every key has lo_d <= k_d <= hi_d, so
//     q.k = sum_d q_d k_d <= sum_d q_d * (q_d > 0 ? hi_d : lo_d),
// and a kv head's score of a block is the largest such bound over the group's query heads. The m highest scores are taken,
// ties to the lower block. The scores are held in f64: q (24 bits) times a bound (11 bits) is exact there, the sum of up to
// 128 of them is off by 2^-46 of its terms, so two blocks change places only where their bounds are equal to that; in f32
// the order of near neighbours (their distance shrinks with the number of blocks) would hang on the order of the sum.
//
// One cluster of CTAs per (row, kv head): the CTAs share out the blocks, 16 (head_dim 128) or 8 (64) lanes to a block with
// eight dims each, and send the scores to the first CTA's shared memory, which selects: a histogram of the scores' range
// in 2048 bins finds the bin of the m-th score, its range is divided again until the bin holds exactly what is
// still needed (or equal scores), and one ordered pass writes the list.
#include "paged.cuh"

namespace {

constexpr int kSelThreads = 256;
constexpr int kSelMaxBlocks = 24576;  // 8 bytes a score in the first CTA's shared memory
constexpr int kSelMaxList = 2048;
constexpr int kSelBins = 2048;

// order-preserving key of a finite score
__device__ __forceinline__ unsigned long long key_of(double s) {
    const long long b = __double_as_longlong(s);
    return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | 0x8000000000000000ull;
}

template <typename T, typename F>
__device__ __forceinline__ T block_fold(T v, T* red, F f) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    T t = red[0];
    for (int w = 1; w < kSelThreads / 32; w++) t = f(t, red[w]);
    return t;
}

// exclusive scan over the block's threads; total in `total`
__device__ __forceinline__ int block_scan(int v, int* red, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
    }
    __syncthreads();
    if (lane == 31) red[warp] = s;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < kSelThreads / 32; w++) {
        if (w < warp) before += red[w];
        total += red[w];
    }
    return before + s - v;
}

template <int HD, int G>
__global__ void __launch_bounds__(kSelThreads) paged_select_kernel(const b200_paged_cache c, const int32_t* __restrict__ row_slot,
                                                                   const int32_t* __restrict__ row_pos, const float* __restrict__ q, size_t ldq,
                                                                   int n_first, int n_recent, int n_select, int32_t* __restrict__ sel) {
    extern __shared__ __align__(16) unsigned long long sel_smem[];  // keys of the middle blocks (first CTA)
    __shared__ unsigned hist[kSelBins];
    __shared__ unsigned long long red_u[kSelThreads / 32];
    __shared__ int red_i[kSelThreads / 32];
    __shared__ int s_bin, s_above, s_in;
    const int ctas = (int)cluster_size(), rank = (int)cluster_rank(), tid = threadIdx.x;
    const int r = blockIdx.x / ctas, kvh = blockIdx.y;
    const int slot = row_slot[r], pos = row_pos[r];
    if (!paged_row_ok(slot, pos, c.n_seqs)) return;  // the whole cluster leaves; the row's list stays as it was
    int32_t* out = sel + ((size_t)r * c.n_kv_heads + kvh) * n_select;
    const int have = paged_visible(pos, c.block_rows, c.max_blocks);
    if (have <= n_select) {
        if (rank == 0)
            for (int i = tid; i < n_select; i += kSelThreads) out[i] = i < have ? i : -1;
        return;
    }
    const int n = have - n_first - n_recent;  // the middle blocks n_first .. n_first + n - 1
    const int m = n_select - n_first - n_recent;
    const int32_t* tbl = c.block_table + (size_t)slot * c.max_blocks + n_first;
    cluster_sync();  // the first CTA has started: its shared memory may be written
    if (m > 0) {
        constexpr int LPB = HD / 8, BPW = 32 / LPB;  // lanes a block, blocks a warp pass
        const int lane = tid & 31, sub = lane % LPB;
        double qd[G][8];
#pragma unroll
        for (int g = 0; g < G; g++) {
            const float* qp = q + (size_t)r * ldq + (size_t)(kvh * G + g) * HD + 8 * sub;
#pragma unroll
            for (int d = 0; d < 8; d++) qd[g][d] = (double)qp[d];
        }
        const unsigned keys0 = cluster_addr(sel_smem, 0);
        const int per = BPW * (kSelThreads / 32) * ctas;
        for (int b0 = (rank * (kSelThreads / 32) + (tid >> 5)) * BPW; b0 < n; b0 += per) {
            const int b = b0 + lane / LPB;
            const int page = b < n ? tbl[b] : 0;
            const bool ok = paged_block_ok(page, c.n_blocks);
            uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
            if (ok) {
                const uint4* p = reinterpret_cast<const uint4*>(static_cast<const __half*>(c.key_bounds) + ((size_t)page * c.n_kv_heads + kvh) * 2 * HD);
                lo = p[sub];
                hi = p[LPB + sub];
            }
            double s[G];
#pragma unroll
            for (int g = 0; g < G; g++) s[g] = 0.0;
            const __half* lh = reinterpret_cast<const __half*>(&lo);
            const __half* hh = reinterpret_cast<const __half*>(&hi);
#pragma unroll
            for (int d = 0; d < 8; d++) {
                const double l = (double)__half2float(lh[d]), u = (double)__half2float(hh[d]);
#pragma unroll
                for (int g = 0; g < G; g++) s[g] = fma(qd[g][d], qd[g][d] > 0.0 ? u : l, s[g]);
            }
#pragma unroll
            for (int o = LPB / 2; o > 0; o >>= 1)
#pragma unroll
                for (int g = 0; g < G; g++) s[g] += __shfl_xor_sync(0xffffffffu, s[g], o);
            constexpr double top = 1.7976931348623157e308;
            double best = -INFINITY;
            bool nan = false;
#pragma unroll
            for (int g = 0; g < G; g++) {
                nan |= s[g] != s[g];
                best = fmax(best, s[g]);
            }
            best = nan ? top : fmin(fmax(best, -top), top) + 0.0;  // -0 -> +0
            if (!ok) best = -top;
            if (sub == 0 && b < n) cluster_store_u64(keys0 + 8u * (unsigned)b, key_of(best));
        }
    }
    cluster_sync();  // the scores are in the first CTA's shared memory
    if (rank != 0) return;

    for (int i = tid; i < n_first; i += kSelThreads) out[i] = i;
    for (int i = tid; i < n_recent; i += kSelThreads) out[n_select - n_recent + i] = have - n_recent + i;
    if (m <= 0) return;
    const unsigned long long* key = sel_smem;
    unsigned long long kmin = ~0ull, kmax = 0;
    for (int i = tid; i < n; i += kSelThreads) {
        kmin = min(kmin, key[i]);
        kmax = max(kmax, key[i]);
    }
    auto lower = [](unsigned long long x, unsigned long long y) { return x < y ? x : y; };
    auto upper = [](unsigned long long x, unsigned long long y) { return x < y ? y : x; };
    kmin = block_fold(kmin, red_u, lower);
    kmax = block_fold(kmax, red_u, upper);
    // every key above `kmax` is taken, none below `kmin`; `need` of those between are
    int need = m;
    while (true) {
        const int width = 64 - __clzll((long long)(kmax - kmin));  // bits of the range
        const int shift = width > 11 ? width - 11 : 0;
        for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kSelThreads) {
            const unsigned long long k = key[i];
            if (k >= kmin && k <= kmax) atomicAdd(&hist[(unsigned)((k - kmin) >> shift)], 1u);
        }
        __syncthreads();
        // thread t holds bins 2047 - 8t down to 2040 - 8t; the bin where the running count reaches `need` is in one of them
        constexpr int BPT = kSelBins / kSelThreads;
        int mine = 0;
        for (int j = 0; j < BPT; j++) mine += (int)hist[kSelBins - 1 - (tid * BPT + j)];
        int total;
        int above = block_scan(mine, red_i, total);
        if (above < need && above + mine >= need) {
            for (int j = 0; j < BPT; j++) {
                const int bin = kSelBins - 1 - (tid * BPT + j), here = (int)hist[bin];
                if (above + here >= need) {
                    s_bin = bin;
                    s_above = above;
                    s_in = here;
                    break;
                }
                above += here;
            }
        }
        __syncthreads();
        const int bin = s_bin, here = s_in;
        need -= s_above;
        const unsigned long long lo = kmin + ((unsigned long long)bin << shift);
        const unsigned long long hi = lo + ((1ull << shift) - 1ull);
        kmax = hi < kmax ? hi : kmax;
        kmin = lo;
        __syncthreads();
        if (here == need || shift == 0) break;
    }
    // keys above kmax are taken, and the first `need` of those from kmin to kmax: all of them, or equal ones by index
    const int per = (n + kSelThreads - 1) / kSelThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    int n_above = 0, n_edge = 0;
    for (int i = i0; i < i1; i++) {
        n_above += key[i] > kmax;
        n_edge += key[i] >= kmin && key[i] <= kmax;
    }
    int total;
    const int above0 = block_scan(n_above, red_i, total);
    int edge = block_scan(n_edge, red_i, total);
    int at = n_first + above0 + min(edge, need);
    for (int i = i0; i < i1; i++) {
        const bool is_edge = key[i] >= kmin && key[i] <= kmax;
        if (key[i] > kmax || (is_edge && edge < need)) out[at++] = n_first + i;
        edge += is_edge;
    }
}

template <int HD>
auto select_kernel(int G) {
    switch (G) {
        case 1: return paged_select_kernel<HD, 1>;
        case 2: return paged_select_kernel<HD, 2>;
        case 3: return paged_select_kernel<HD, 3>;
        case 4: return paged_select_kernel<HD, 4>;
        case 5: return paged_select_kernel<HD, 5>;
        case 6: return paged_select_kernel<HD, 6>;
        case 7: return paged_select_kernel<HD, 7>;
        default: return paged_select_kernel<HD, 8>;
    }
}

}  // namespace

extern "C" int b200_paged_select(b200_ctx* ctx, const b200_paged_cache* c, const b200_paged_rows* r, const float* q, int ldq, int n_heads, int n_first,
                                 int n_recent, int n_select, int32_t* sel) {
    if (!ctx) return B200_BAD_ARGUMENT;
    PagedNeeds need;
    need.bounds = true;
    ST_TRY(paged_check(ctx, "b200_paged_select", c, r, need));
    if (n_heads < 1 || n_heads % c->n_kv_heads || n_heads / c->n_kv_heads > 8)
        B200_FAIL(ctx, B200_BAD_ARGUMENT, "b200_paged_select: %d query heads over %d kv heads; a group has 1 to 8 query heads", n_heads, c->n_kv_heads);
    if (n_first < 0 || n_recent < 1 || n_select < 1 || n_select > kSelMaxList || n_first > n_select - n_recent)
        B200_FAIL(ctx, B200_BAD_ARGUMENT, "b200_paged_select: %d blocks with the first %d and the last %d; 1 to %d blocks, the last one among them", n_select,
                  n_first, n_recent, kSelMaxList);
    if (c->max_blocks > kSelMaxBlocks)
        B200_FAIL(ctx, B200_BAD_ARGUMENT, "b200_paged_select: %d table entries; scores of at most %d blocks fit a CTA's shared memory", c->max_blocks, kSelMaxBlocks);
    if (r->n_rows == 0) return B200_OK;
    if (!q || !sel || paged_misaligned(q, 16) || paged_misaligned(sel, 4) || ldq < (long long)n_heads * c->head_dim || (ldq & 3))
        B200_FAIL(ctx, B200_BAD_ARGUMENT, "b200_paged_select: q must be 16-byte aligned with a stride of at least n_heads * head_dim floats, a multiple of 4; "
                                          "sel 4-byte aligned (got a stride of %d)", ldq);
    if (c->n_kv_heads > 65535) B200_FAIL(ctx, B200_BAD_ARGUMENT, "b200_paged_select: %d kv heads", c->n_kv_heads);
    if (ctx->device < 0) B200_FAIL(ctx, B200_CUDA_ERROR, "b200_paged_select: the context has no device");
    DeviceScope dev;
    CUDA_TRY(ctx, dev.enter(ctx->device));
    const int G = n_heads / c->n_kv_heads;
    auto kernel = c->head_dim == 128 ? select_kernel<128>(G) : select_kernel<64>(G);
    static SmemLimit limit[2][8];
    const size_t smem = 8 * (size_t)c->max_blocks;
    CUDA_TRY(ctx, limit[c->head_dim == 128][G - 1].raise(kernel, ctx->device, 8 * (size_t)kSelMaxBlocks));
    int ctas = 1;
    while (ctas < 8 && (long long)r->n_rows * c->n_kv_heads * ctas < 2 * ctx->sm_count && c->max_blocks / ctas > 64) ctas *= 2;
    launch_cluster(kernel, ctas, dim3((unsigned)(r->n_rows * ctas), c->n_kv_heads), dim3(kSelThreads), smem, ctx->stream, *c, r->row_slot, r->row_pos, q,
                   (size_t)ldq, n_first, n_recent, n_select, sel);
    LAUNCH_CHECK(ctx);
    return B200_OK;
}
