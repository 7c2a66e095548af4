// paged_select.cu — which blocks of a long context a query should attend (b200_paged_select).
//
// A block's key bounds give an upper bound of q.k over its keys: every key has lo_d <= k_d <= hi_d, so
//     q.k = sum_d q_d k_d <= s_g = sum_d q_d * (q_d > 0 ? hi_d : lo_d),
// and a kv head's score of a block is the largest s_g over the group's query heads. The m highest scores are taken, ties to
// the lower block. The order is that of the scores in f64: q (24 bits) times a bound (11 bits) is exact there and the sum
// of up to 128 of them is off by 2^-46 of its terms; in f32 the order of near neighbours would hang on the order of the sum.
//
// Reading the bounds once is what the call cannot do without (4 HD bytes a block and kv head), and f64 for every block would
// cost more than that (f64 multiply-adds and conversions for G heads: 220 us for 256 rows of 32/8 heads of 128 over 260
// blocks each, where the bytes take 42). So the scores are first taken on the matrix unit, with a bound of their error:
//     s~ = sum_{q > 0} q_d hi_d + sum_{q <= 0} q_d lo_d     as mma.sync m16n8k16: 16 blocks x 8 heads x 16 dims,
// q scaled by a power of two (largest |q| in [1, 2)) and split into fp16 parts hi + 2^-11 lo, products exact, fp32 sums. The
// split leaves at most 2^-22 |q_d| or 2^-36. No document says how the unit rounds; assumed is that a step which adds 16 products to the
// sum is off by at most 17 * 2^-23 of the terms' absolute sum S, one unit in the last place for each term cut off (observed: 2.3 * 2^-23 at
// most, over 12 million steps with terms alike, of one sign, and 2^56 apart), and the eight steps of either sum by 2^-15.9 S.
// E = 2^-14 S + 2^-12 covers it (128 dims of the largest fp16 bound times 2^-36 are 2^-13), with S = sum |q_d| max(|lo_d|, |hi_d|), which is
// no less than the terms' sum, from the same unit. The true m-th
// score lies within E of the m-th s~, so a block whose s~ is more than 2E above (below) that is in (out) for certain; only
// the blocks between (a handful) are scored in f64. An infinity or a NaN anywhere makes E infinite, and every block is
// scored in f64.
//
// One cluster of CTAs per (row, kv head). Each CTA scores a run of the blocks, keeps its s~ in shared memory and decides about
// its own blocks; what the cluster has to agree on goes through distributed shared memory, every CTA reading the same: the
// range of s~ and E, a histogram in 512 bins that finds the bin of the m-th (taken again inside the bin where that is much
// wider than E), and the f64 scores of the blocks in doubt. A bit per block says which are in; an ordered pass over the
// words of bits writes the list. Where the scores are few enough for one CTA, the first one gathers them and does all of
// that alone.
#include "paged.cuh"

namespace {

constexpr int kSelThreads = 128, kSelWarps = kSelThreads / 32;
constexpr int kSelMaxBlocks = 24576;  // a CTA that is alone holds a score and two bits for each in shared memory
constexpr int kSelMaxList = 2048;
constexpr int kSelBins = 512;         // four a thread
constexpr int kSelDoubt = 256;        // blocks in doubt that are ranked in a list; more are selected among in place
constexpr int kSelMaxCluster = 8;
constexpr int kSelGather = 512;       // room for as many scores costs a CTA little, and the choice among them is quick
constexpr int kSelRun = 16 * kSelWarps;  // blocks a CTA scores at a time
// Dynamic shared memory with which four CTAs fit the 228 KB of an SM, and with which three do but not four (head_dim 64, 128). A CTA
// has 12 to 14 KB of static shared memory, or 17 to 21, and 1 KB that the system keeps. Three stay within 196 KB, so that the L1
// cache keeps 60: at 208 KB it has 28, and what a row's loads share no longer stays in it (head_dim 128, a group of 8, 320 pairs
// of 500 blocks 38 against 26 us).
constexpr size_t kSelFour = 35 * 1024, kSelThree[2] = {46 * 1024, 40 * 1024};

__device__ __forceinline__ void mma16816(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A load that stays where it is written: all of a run's loads go out before its first product waits for one.
__device__ __forceinline__ uint4 load16(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ unsigned half2_bits(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const unsigned*>(&h);
}

// order-preserving key of a finite f64 score
__device__ __forceinline__ unsigned long long key_of(double s) {
    const long long b = __double_as_longlong(s);
    return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | 0x8000000000000000ull;
}

// Finds the bin in which the running count from the top of the cluster's histogram (the sum of the CTAs') reaches `need`, and
// the counts above it and in it. A thread holds four bins.
struct Found {
    int bin, above, in;
};
__device__ __forceinline__ void find_bin(const unsigned* hist, int ctas, int need, int* red, Found* found) {
    constexpr int BPT = kSelBins / kSelThreads;
    static_assert(BPT == 4, "a uint4 a thread");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = kSelBins - BPT * (1 + (int)threadIdx.x);
    uint4 h = make_uint4(0, 0, 0, 0);
    if (ctas == 1) {
        h = *reinterpret_cast<const uint4*>(hist + first);
    } else {
        uint4 t[kSelMaxCluster];
#pragma unroll
        for (int w = 0; w < kSelMaxCluster; w++) t[w] = w < ctas ? cluster_load_u32x4(cluster_addr(hist + first, w)) : h;
#pragma unroll
        for (int w = 0; w < kSelMaxCluster; w++) { h.x += t[w].x; h.y += t[w].y; h.z += t[w].z; h.w += t[w].w; }
    }
    const int count[BPT] = {(int)h.w, (int)h.z, (int)h.y, (int)h.x};  // from the top
    const int mine = count[0] + count[1] + count[2] + count[3];
    int above = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, above, o);
        if (lane >= o) above += t;
    }
    if (lane == 31) red[warp] = above;
    __syncthreads();
    above -= mine;
#pragma unroll
    for (int w = 0; w < kSelWarps; w++) above += w < warp ? red[w] : 0;
    if (above < need && above + mine >= need) {
#pragma unroll
        for (int j = 0; j < BPT; j++) {
            if (above < need && above + count[j] >= need) {
                *found = Found{first + BPT - 1 - j, above, count[j]};
                above = need;  // found
            } else {
                above += count[j];
            }
        }
    }
    __syncthreads();
}

// Key of the f64 score of one block by the HD/8 lanes that share it (eight dims each, `sub` among them); every lane gets it.
// The order of summation is the same for every block, so equal bounds have equal scores.
template <int HD>
__device__ __forceinline__ unsigned long long exact_key(const b200_paged_cache& c, int page, int kvh, const float* q, int G, int sub) {
    constexpr int LPB = HD / 8;
    constexpr double top = 1.7976931348623157e308;
    const bool ok = paged_block_ok(page, c.n_blocks);
    uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
    if (ok) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const __half*>(c.key_bounds) + ((size_t)page * c.n_kv_heads + kvh) * 2 * HD);
        lo = p[sub];
        hi = p[LPB + sub];
    }
    const __half* lh = reinterpret_cast<const __half*>(&lo);
    const __half* hh = reinterpret_cast<const __half*>(&hi);
    double best = -INFINITY;
    bool nan = false;
#pragma unroll 4
    for (int g = 0; g < G; g++) {
        const float4 a = *reinterpret_cast<const float4*>(q + g * HD + 8 * sub), b = *reinterpret_cast<const float4*>(q + g * HD + 8 * sub + 4);
        const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        double s = 0.0, t = 0.0;
#pragma unroll
        for (int d = 0; d < 8; d += 2) {
            s = fma((double)x[d], (double)__half2float(x[d] > 0.f ? hh[d] : lh[d]), s);
            t = fma((double)x[d + 1], (double)__half2float(x[d + 1] > 0.f ? hh[d + 1] : lh[d + 1]), t);
        }
        s += t;
#pragma unroll
        for (int o = LPB / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        nan |= s != s;
        best = fmax(best, s);
    }
    best = nan ? top : fmin(fmax(best, -top), top) + 0.0;  // -0 -> +0
    return key_of(ok ? best : -top);
}

// Four CTAs an SM: the 128 registers this leaves a thread hold a run's bounds (64) on their way; left to itself the compiler takes
// fewer and starts the products before the last load is out (batch 66.5 against 57.6 us, long contexts 59.9 against 47.1 us).
template <int HD, bool NARROW>
__global__ void __launch_bounds__(kSelThreads, 4) paged_select_kernel(const b200_paged_cache c, const int32_t* row_slot,
                                                                   const int32_t* row_pos, const float* q, size_t ldq, int G,
                                                                   int n_first, int n_recent, int n_select, int max_chunk, int32_t* sel) {
    pdl_wait();
    // the CTA's blocks: s~ (with many blocks in doubt, words of their keys), a bit for those that are in, one for those in doubt
    extern __shared__ __align__(16) float sel_score[];
    unsigned* in_bits = reinterpret_cast<unsigned*>(sel_score + max_chunk);
    unsigned* doubt_bits = in_bits + max_chunk / 32;
    __shared__ __align__(16) unsigned hist[kSelBins];
    __shared__ __align__(16) float sq[8][HD];
    __shared__ __align__(16) uint4 q_frag[HD / 32][NARROW ? 3 : 5][32];  // chunk of dims, part (q > 0, q <= 0, |q|; their lo), lane
    // what the CTAs tell one another, by rank (and warp)
    __shared__ __align__(16) float s_err[kSelMaxCluster * kSelWarps], s_min[kSelMaxCluster * kSelWarps], s_max[kSelMaxCluster * kSelWarps];
    __shared__ unsigned s_word[kSelMaxCluster * kSelWarps], s_top[kSelMaxCluster * kSelWarps];
    __shared__ int n_in[kSelMaxCluster], n_doubt_of[kSelMaxCluster], n_left[kSelMaxCluster], n_taken[kSelMaxCluster];
    __shared__ unsigned long long doubt_key[kSelDoubt];  // the cluster's blocks in doubt: score and block
    __shared__ int doubt[kSelDoubt];
    __shared__ int own_doubt[kSelDoubt];
    __shared__ int red_i[kSelWarps];
    __shared__ Found found;
    __shared__ int s_in, s_doubt;  // this CTA's blocks that are in for certain and in doubt
    int ctas = (int)cluster_size();
    const int rank = (int)cluster_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = blockIdx.x / ctas, kvh = blockIdx.y;
    const int slot = row_slot[r], pos = row_pos[r];
    const float* qr = q + (size_t)r * ldq + (size_t)kvh * G * HD;
    float4 q_ahead[8 * HD / (4 * kSelThreads)];  // on its way beside the row's place
#pragma unroll
    for (int i = 0; i < 8 * HD / (4 * kSelThreads); i++)
        q_ahead[i] = tid + i * kSelThreads < G * HD / 4 ? reinterpret_cast<const float4*>(qr)[tid + i * kSelThreads] : make_float4(0.f, 0.f, 0.f, 0.f);
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
    const int32_t* tbl = c.block_table + (size_t)slot * c.max_blocks + n_first;  // of this CTA's blocks from below on
    if (rank == 0) {
        for (int i = tid; i < n_first; i += kSelThreads) out[i] = i;
        for (int i = tid; i < n_recent; i += kSelThreads) out[n_select - n_recent + i] = have - n_recent + i;
    }
    if (m <= 0) return;
    auto everyone = [&] {
        if (ctas > 1) cluster_sync(); else __syncthreads();
    };
    auto tell = [&](auto* what, auto v) {  // a warp's first lanes: one CTA each
        if (lane < ctas) cluster_store(cluster_addr(what, lane), v);
    };
    if (ctas > 1) cluster_arrive();
    auto clear = [&] {
        for (int i = 4 * tid; i < kSelBins; i += 4 * kSelThreads) *reinterpret_cast<uint4*>(hist + i) = make_uint4(0, 0, 0, 0);
    };
    clear();
    if (tid == 0) s_in = s_doubt = 0;
    // this CTA's blocks: from .. from + own - 1 of the middle, 16 a warp at a time
    const int chunk = (n + kSelRun * ctas - 1) / (kSelRun * ctas) * kSelRun, from = min(n, rank * chunk);
    int own = min(n, from + chunk) - from;
    tbl += from;
    // few enough for one CTA: the first one gathers the scores and chooses alone, without another cluster barrier
    const bool gather = ctas > 1 && n <= max_chunk;
    {
        // Fragments: row of A = block, column of B = head. A lane's words of a 16-byte chunk are taken as the dims of its
        // places in the k steps; q is laid out by the same rule, so a bound is loaded as it lies. With up to four heads (NARROW)
        // columns 0 .. 3 hold the parts hi of q and 4 .. 7 the parts lo, else lo takes products of its own.
        constexpr int CH = HD / 32;  // 16-byte chunks of a row per lane: chunks tig, tig + 4, ...
        constexpr unsigned abs2 = 0x7fff7fffu;
        const int gid = lane >> 2, tig = lane & 3;
        int b0 = 16 * warp;
        auto page_of = [&](int b) { return b < own ? tbl[b] : 0; };
        int page0 = page_of(b0 + gid), page1 = page_of(b0 + 8 + gid);
#pragma unroll
        for (int i = 0; i < 8 * HD / (4 * kSelThreads); i++) reinterpret_cast<float4*>(&sq[0][0])[tid + i * kSelThreads] = q_ahead[i];
        __syncthreads();
        // the columns' powers of two against the group's largest; columns past the group repeat its first head
        float f0, f1;
        {
            const int head = NARROW ? gid & 3 : gid;
            const float* qp = sq[head < G ? head : 0] + 8 * tig;
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < 2 * CH; i++) {
                const float4 u = *reinterpret_cast<const float4*>(qp + 32 * (i >> 1) + 4 * (i & 1));
                most = fmaxf(fmaxf(most, fmaxf(fabsf(u.x), fabsf(u.y))), fmaxf(fabsf(u.z), fabsf(u.w)));
            }
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            // the head's largest |q| comes to [1, 2); 2^-126 and less count as 2^-126 (the floor of E covers them)
            const int e = max(-126, min(127, (int)(__float_as_uint(most) >> 23) - 127));
            const float down0 = pow2(-(e / 2)), down1 = pow2(-(e - e / 2));  // 2^-e in two factors, each of them normal
            int e_max = e;
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) e_max = max(e_max, __shfl_xor_sync(0xffffffffu, e_max, o));
            const float f = pow2(max(-126, e - e_max));
            f0 = __shfl_sync(0xffffffffu, f, 8 * tig);  // of column 2 tig: that column's lanes hold its head's factor
            f1 = __shfl_sync(0xffffffffu, f, 8 * tig + 4);
            auto split = [](float a, float b, unsigned& hi, unsigned& lo) {
                hi = half2_bits(a, b);
                const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                lo = half2_bits((a - t.x) * 2048.f, (b - t.y) * 2048.f);
            };
            if (warp < CH) {  // each warp lays out one chunk of the dims; word j of a part: dims 2j, 2j + 1 of the lane's eight
                const float4 u = *reinterpret_cast<const float4*>(qp + 32 * warp), v = *reinterpret_cast<const float4*>(qp + 32 * warp + 4);
                const float x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
                unsigned w[5][4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float a = x[2 * j] * down0 * down1, b = x[2 * j + 1] * down0 * down1;
                    // !(q > 0) goes with the lower bounds, a NaN as well
                    split(a > 0.f ? a : 0.f, b > 0.f ? b : 0.f, w[0][j], w[3][j]);
                    split(a > 0.f ? 0.f : a, b > 0.f ? 0.f : b, w[1][j], w[4][j]);
                    w[2][j] = w[0][j] | (w[1][j] & abs2);
                    if (NARROW && gid >= 4) {
                        w[0][j] = w[3][j];
                        w[1][j] = w[4][j];
                    }
                }
#pragma unroll
                for (int t = 0; t < (NARROW ? 3 : 5); t++) q_frag[warp][t][lane] = make_uint4(w[t][0], w[t][1], w[t][2], w[t][3]);
            }
        }
        __syncthreads();
        // E is never negative, so its bits order as it does, and an infinity or a NaN (0 * inf) is above every number
        unsigned err_bits = 0;
        float mn = INFINITY, mx = -INFINITY;
        const float k0 = 0x1p-14f * f0, k1 = 0x1p-14f * f1, floor0 = 0x1p-12f * f0, floor1 = 0x1p-12f * f1;
        const uint8_t* bounds = static_cast<const uint8_t*>(c.key_bounds) + (size_t)kvh * 4 * HD + 16 * tig;
        const size_t block_bytes = (size_t)c.n_kv_heads * 4 * HD;
        for (; b0 < own; b0 += kSelRun) {
            const bool ok0 = paged_block_ok(page0, c.n_blocks), ok1 = paged_block_ok(page1, c.n_blocks);
            // (what is not mapped is read from the null block and does not count)
            const uint8_t *p0 = bounds + (ok0 ? page0 : 0) * block_bytes, *p1 = bounds + (ok1 ? page1 : 0) * block_bytes;
            uint4 l0[CH], l1[CH], h0[CH], h1[CH];
#pragma unroll
            for (int i = 0; i < CH; i++) {
                h0[i] = load16(p0 + 2 * HD + 64 * i);
                h1[i] = load16(p1 + 2 * HD + 64 * i);
                l0[i] = load16(p0 + 64 * i);
                l1[i] = load16(p1 + 64 * i);
            }
            page0 = page_of(b0 + kSelRun + gid);
            page1 = page_of(b0 + kSelRun + 8 + gid);
            float up[4] = {0, 0, 0, 0}, dn[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0}, sum[4] = {0, 0, 0, 0};
            // two k steps on a chunk of the bounds: words 0, 1 and words 2, 3
            auto product = [](float (&c)[4], const uint4& a, const uint4& b, const uint4& q) {
                mma16816(c, a.x, b.x, a.y, b.y, q.x, q.y);
                mma16816(c, a.z, b.z, a.w, b.w, q.z, q.w);
            };
            auto larger = [](const uint4& a, const uint4& b) {  // of the magnitudes; a NaN stays
                return make_uint4(max_nan2(a.x & abs2, b.x & abs2), max_nan2(a.y & abs2, b.y & abs2), max_nan2(a.z & abs2, b.z & abs2),
                                  max_nan2(a.w & abs2, b.w & abs2));
            };
#pragma unroll
            for (int i = 0; i < CH; i++) {
                product(up, h0[i], h1[i], q_frag[i][0][lane]);
                product(dn, l0[i], l1[i], q_frag[i][1][lane]);
                product(sum, larger(h0[i], l0[i]), larger(h1[i], l1[i]), q_frag[i][2][lane]);
                if constexpr (!NARROW) {
                    product(lo, h0[i], h1[i], q_frag[i][3][lane]);
                    product(lo, l0[i], l1[i], q_frag[i][4][lane]);
                }
            }
            // columns 2 tig and 2 tig + 1 of rows gid (values 0, 1) and gid + 8 (values 2, 3)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const bool ok = h ? ok1 : ok0;
                const int b = b0 + 8 * h + gid;
                const float E0 = fmaf(sum[2 * h], k0, floor0), E1 = fmaf(sum[2 * h + 1], k1, floor1);
                float hi0 = up[2 * h] + dn[2 * h], hi1 = up[2 * h + 1] + dn[2 * h + 1], lo0 = lo[2 * h], lo1 = lo[2 * h + 1];
                if constexpr (NARROW) {  // the same head's other part is two lanes away
                    const float other0 = __shfl_xor_sync(0xffffffffu, hi0, 2), other1 = __shfl_xor_sync(0xffffffffu, hi1, 2);
                    lo0 = tig < 2 ? other0 : hi0;
                    lo1 = tig < 2 ? other1 : hi1;
                    hi0 = tig < 2 ? hi0 : other0;
                    hi1 = tig < 2 ? hi1 : other1;
                }
                float s = fmaxf(fmaf(lo0, 0x1p-11f, hi0) * f0, fmaf(lo1, 0x1p-11f, hi1) * f1);
                s = fmaxf(s, __shfl_xor_sync(0xffffffffu, s, 1));
                if constexpr (!NARROW) s = fmaxf(s, __shfl_xor_sync(0xffffffffu, s, 2));
                if (ok) {
                    err_bits = max(err_bits, max(__float_as_uint(E0) & 0x7fffffffu, __float_as_uint(E1) & 0x7fffffffu));
                    mn = fminf(mn, s);
                    mx = fmaxf(mx, s);
                }
                if (tig == 0 && b < own) sel_score[b] = ok ? s : -INFINITY;
            }
        }
        pdl_trigger();
        err_bits = __reduce_max_sync(0xffffffffu, err_bits);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        }
        const float err = __uint_as_float(min(err_bits, 0x7f800000u));
        if (ctas > 1) cluster_wait();  // the CTAs have started: their shared memory may be written
        if (gather && rank > 0) {
            __syncthreads();
            const unsigned there = cluster_addr(sel_score + from, 0);
            for (int i = 4 * tid; i < own; i += 4 * kSelThreads) cluster_store(there + 4u * (unsigned)i, *reinterpret_cast<const float4*>(sel_score + i));
        }
        const int at = rank * kSelWarps + warp;
        tell(s_err + at, err);
        tell(s_min + at, mn);
        tell(s_max + at, mx);
    }
    everyone();

    const int told = ctas * kSelWarps;
    if (gather) {
        if (rank > 0) return;
        ctas = 1;
        own = n;
    }
    float err = 0.f, lo = INFINITY, hi = -INFINITY;
    static_assert(kSelWarps == 4, "a CTA's figures are read as one float4");
    for (int i = 0; i < told; i += 4) {
        const float4 e = *reinterpret_cast<const float4*>(s_err + i), a = *reinterpret_cast<const float4*>(s_min + i), b = *reinterpret_cast<const float4*>(s_max + i);
        err = fmaxf(err, fmaxf(fmaxf(e.x, e.y), fmaxf(e.z, e.w)));
        lo = fminf(lo, fminf(fminf(a.x, a.y), fminf(a.z, a.w)));
        hi = fmaxf(hi, fmaxf(fmaxf(b.x, b.y), fmaxf(b.z, b.w)));
    }
    err *= 1.01f;  // what the comparisons below round
    // [lo, hi] holds the m-th largest s~. Unmapped blocks count as the least s~: too much, but never enough to be in for certain.
    if (!(lo <= hi)) lo = hi = 0.f;  // nothing is mapped
    const float floor_s = lo;
    auto score = [&](int i) { return fmaxf(sel_score[i], floor_s); };
    if (err < INFINITY) {
        for (int pass = 0; pass < 3 && hi - lo > 16.f * err; pass++) {
            // s~ above the range (from the second pass on) counts in the top bin: the m-th lies in the range, so its bin is found
            const float range = hi - lo, inv = __fdividef((float)(kSelBins - 1), range), width = range * (1.f / (kSelBins - 1));
#pragma unroll 4
            for (int i = tid; i < own; i += kSelThreads) {
                const float s = score(i);
                if (s >= lo) atomicAdd(&hist[min(kSelBins - 1, (int)((fminf(s, hi) - lo) * inv))], 1u);
            }
            everyone();
            find_bin(hist, ctas, m, red_i, &found);
            // the bin's edges, out by more than the index above and they themselves round (2^-21 of the range)
            const float slack = range * 0x1p-19f, from_s = fmaf((float)found.bin, width, lo) - slack, to_s = fmaf((float)(found.bin + 1), width, lo) + slack;
            lo = fmaxf(lo, from_s);
            hi = fminf(hi, to_s);
            if (hi - lo > 16.f * err) {
                everyone();  // the histograms have been read
                clear();
                __syncthreads();
            }
        }
    } else {
        lo = -INFINITY;
        hi = INFINITY;
    }
    // in for certain, out for certain, in doubt
    const float sure_in = hi + 2.f * err, sure_out = lo - 2.f * err;
    const int words = (own + 31) >> 5;
    int in = 0;
#pragma unroll 2
    for (int w = warp; w < words; w += kSelWarps) {
        const int i = 32 * w + lane;
        const float s = i < own ? score(i) : -INFINITY;
        const bool is_in = i < own && s > sure_in, is_doubt = i < own && !(s > sure_in) && !(s < sure_out);
        const unsigned in_word = __ballot_sync(0xffffffffu, is_in), doubt_word = __ballot_sync(0xffffffffu, is_doubt);
        if (doubt_word) {
            int at = lane == 0 ? atomicAdd(&s_doubt, __popc(doubt_word)) : 0;
            at = __shfl_sync(0xffffffffu, at, 0) + __popc(doubt_word & ((1u << lane) - 1u));
            if (is_doubt && at < kSelDoubt) own_doubt[at] = i;
        }
        if (lane == 0) {
            in_bits[w] = in_word;
            doubt_bits[w] = doubt_word;
        }
        in += __popc(in_word);
    }
    if (lane == 0 && in > 0) atomicAdd(&s_in, in);
    __syncthreads();
    const int n_own = s_doubt;
    int need = m - s_in, n_doubt = n_own, before = 0;  // of the cluster; before: blocks in doubt of the CTAs ahead
    int first = n_first;                               // this CTA's first place in the list
    if (ctas > 1) {
        if (warp == 0) {
            tell(n_in + rank, s_in);
            tell(n_doubt_of + rank, n_own);
        }
        everyone();
        need = m;
        n_doubt = 0;
        for (int w = 0; w < ctas; w++) {
            if (w == rank) {
                before = n_doubt;
                first += m - need;
            }
            need -= n_in[w];
            n_doubt += n_doubt_of[w];
        }
    }
    // `need`, 1 .. n_doubt, of those in doubt are in
    constexpr int LPB = HD / 8, BPW = 32 / LPB;
    const int sub = lane % LPB, part = lane / LPB;
    if (n_doubt == need) {
        for (int w = tid; w < words; w += kSelThreads) in_bits[w] |= doubt_bits[w];
        first += before;
    } else if (n_doubt <= kSelDoubt) {
        for (int j0 = warp * BPW; j0 < n_own; j0 += kSelWarps * BPW) {
            const int j = j0 + part, i = j < n_own ? own_doubt[j] : 0;
            const unsigned long long k = exact_key<HD>(c, j < n_own ? tbl[i] : 0, kvh, &sq[0][0], G, sub);
            if (j < n_own && sub < ctas) {  // (a cluster has at most as many CTAs as a block has lanes)
                cluster_store(cluster_addr(doubt_key + before + j, sub), k);
                cluster_store(cluster_addr(doubt + before + j, sub), from + i);
            }
        }
        everyone();
        int ahead = 0;  // of those that the CTAs ahead hold, the ones that are in
        for (int j0 = 0; j0 < n_doubt; j0 += kSelThreads) {
            const int j = j0 + tid;
            int higher = n_doubt;
            if (j < n_doubt) {
                const unsigned long long k = doubt_key[j];
                const int i = doubt[j];
                higher = 0;
                for (int t = 0; t < n_doubt; t++) higher += doubt_key[t] > k || (doubt_key[t] == k && doubt[t] < i);
                if (higher < need && j >= before && j < before + n_own) atomicOr(&in_bits[(i - from) >> 5], 1u << ((i - from) & 31));
            }
            ahead += __syncthreads_count(higher < need && j < before);
        }
        first += ahead;
    } else {
        // Equal scores by the hundred, or an infinite E: the upper words of the f64 keys are selected among first, then the
        // lower words of those whose upper word is the last one taken, then the blocks' order decides.
        unsigned* key = reinterpret_cast<unsigned*>(sel_score);
        auto in_doubt = [&](int i) { return ((doubt_bits[i >> 5] >> (i & 31)) & 1u) != 0; };
        for (int level = 0; level < 2 && need > 0; level++) {
            __syncthreads();
            unsigned kmin = ~0u, kmax = 0u;
            for (int i0 = warp * BPW; i0 < own; i0 += kSelWarps * BPW) {
                const int i = i0 + part;
                const bool here = i < own && in_doubt(i);
                if (!__any_sync(0xffffffffu, here)) continue;
                const unsigned long long k = exact_key<HD>(c, here ? tbl[i] : 0, kvh, &sq[0][0], G, sub);
                const unsigned word = level == 0 ? (unsigned)(k >> 32) : (unsigned)k;
                if (here) {
                    if (sub == 0) key[i] = word;
                    kmin = min(kmin, word);
                    kmax = max(kmax, word);
                }
            }
            tell(s_word + rank * kSelWarps + warp, __reduce_min_sync(0xffffffffu, kmin));
            tell(s_top + rank * kSelWarps + warp, __reduce_max_sync(0xffffffffu, kmax));
            everyone();
            for (int i = 0; i < ctas * kSelWarps; i++) {  // (one CTA that gathered tells itself alone)
                kmin = min(kmin, s_word[i]);
                kmax = max(kmax, s_top[i]);
            }
            int here;
            while (true) {  // at most four divisions of the range by 512
                const int width = 32 - __clz((int)(kmax - kmin)), shift = width > 9 ? width - 9 : 0;
                clear();
                __syncthreads();
                for (int i = tid; i < own; i += kSelThreads)
                    if (in_doubt(i) && key[i] >= kmin && key[i] <= kmax) atomicAdd(&hist[(key[i] - kmin) >> shift], 1u);
                everyone();
                find_bin(hist, ctas, need, red_i, &found);
                here = found.in;
                need -= found.above;
                const unsigned edge = kmin + ((unsigned)found.bin << shift), width_less_1 = (1u << shift) - 1u;
                kmax = kmax - edge < width_less_1 ? kmax : edge + width_less_1;  // (edge + width may pass 2^32)
                kmin = edge;
                everyone();  // the histograms have been read
                if (here == need || shift == 0) break;
            }
            // what lies above is in; what lies between is in when all of it is needed, else in doubt still
            const bool all = here == need;
            for (int w = warp; w < words; w += kSelWarps) {
                const int i = 32 * w + lane;
                const bool d = i < own && in_doubt(i);
                const unsigned k = d ? key[i] : 0u;
                const unsigned edge = __ballot_sync(0xffffffffu, d && k >= kmin && k <= kmax), above = __ballot_sync(0xffffffffu, d && k > kmax);
                __syncwarp();
                if (lane == 0) {
                    in_bits[w] |= above | (all ? edge : 0u);
                    doubt_bits[w] = edge;
                }
            }
            if (all) need = 0;
        }
        __syncthreads();
        int left = 0;
        for (int w = lane; w < words; w += 32) left += __popc(doubt_bits[w]);
        left = __reduce_add_sync(0xffffffffu, left);
        if (warp == 0) tell(n_left + rank, left);
        everyone();
        for (int w = 0; w < rank; w++) need -= n_left[w];
        if (tid == 0)  // the first of equals
            for (int w = 0; need > 0 && w < words; w++)
                for (unsigned bits = doubt_bits[w]; bits && need > 0; bits &= bits - 1u, need--) in_bits[w] |= bits & (0u - bits);
        __syncthreads();
        int taken = 0;
        for (int w = lane; w < words; w += 32) taken += __popc(in_bits[w]);
        taken = __reduce_add_sync(0xffffffffu, taken);
        if (warp == 0) tell(n_taken + rank, taken);
        everyone();
        first = n_first;
        for (int w = 0; w < rank; w++) first += n_taken[w];
    }
    __syncthreads();
    // every warp scans the words' counts and writes the blocks of its own words
    for (int g = 0; g < words; g += 32) {
        const unsigned mine = g + lane < words ? in_bits[g + lane] : 0u;
        int end = __popc(mine);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end += t;
        }
        for (int w = warp; w < 32 && g + w < words; w += kSelWarps) {
            const unsigned bits = __shfl_sync(0xffffffffu, mine, w);
            const int at = first + __shfl_sync(0xffffffffu, end, w) - __popc(bits >> lane);
            if (((bits >> lane) & 1u) && at < n_select - n_recent) out[at] = n_first + from + 32 * (g + w) + lane;
        }
        first += __shfl_sync(0xffffffffu, end, 31);
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
    auto kernel = c->head_dim == 128 ? (G <= 4 ? paged_select_kernel<128, true> : paged_select_kernel<128, false>)
                                     : (G <= 4 ? paged_select_kernel<64, true> : paged_select_kernel<64, false>);
    const int variant = 2 * (c->head_dim == 128) + (G <= 4);
    const long long pairs = (long long)r->n_rows * c->n_kv_heads;
    auto chunk_of = [&](int ctas) {  // scores a CTA has room for
        const int chunk = ceil_div(c->max_blocks, kSelRun * ctas) * kSelRun;
        return chunk >= kSelGather ? chunk : c->max_blocks < kSelGather ? ceil_div(c->max_blocks, kSelRun) * kSelRun : kSelGather;
    };
    auto smem_of = [](int blocks) { return (size_t)blocks * 4 + 2 * ((size_t)blocks / 8); };
    static SmemLimit limit[4];
    static ClusterFit fits[4][2], fits_three[4];
    CUDA_TRY(ctx, limit[variant].raise(kernel, ctx->device, smem_of(kSelMaxBlocks)));
    // CTAs a (row, kv head): doubled until there are two an SM, as long as the GPU holds all clusters at once and each CTA has
    // blocks to score. 72 pairs of 500 blocks take 13.3 us as clusters of 8, of which 71 fit, 10.9 as clusters of 4; 144 pairs
    // of 1875 blocks at head_dim 64 33.5 as clusters of 4, 27.2 as pairs.
    int lg = 0;
    for (int fit = 0; (kSelMaxCluster >> lg) > 1 && pairs << lg < 2ll * ctx->sm_count && c->max_blocks > kSelRun << lg; lg++) {
        const bool roomy = smem_of(chunk_of(2 << lg)) > kSelFour;
        CUDA_TRY(ctx, fits[variant][roomy].count(kernel, ctx->device, lg + 1, dim3(kSelThreads), roomy ? smem_of(kSelMaxBlocks / 2) : kSelFour, &fit));
        if (pairs > fit) break;
    }
    // Clusters are placed four to an SM, which with three CTAs for each leaves a quarter of the SMs idle. Where the GPU holds them
    // so, the launch asks for shared memory that keeps a fourth out: 160 pairs of 250 blocks 10.8 -> 9.8 us, of 500 15.1 -> 13.5;
    // 40 pairs of 1875 17.4 -> 15.5; single CTAs, 440 pairs of 1875, 89 -> 79 us.
    const int chunk = chunk_of(1 << lg);
    const size_t three = kSelThree[c->head_dim == 128];
    size_t smem = smem_of(chunk);
    if (pairs << lg > 2ll * ctx->sm_count && smem < three) {
        int fit = 0;
        CUDA_TRY(ctx, fits_three[variant].count(kernel, ctx->device, lg, dim3(kSelThreads), three, &fit));
        if (pairs <= fit) smem = three;
    }
    launch_cluster(kernel, 1 << lg, dim3((unsigned)(r->n_rows << lg), c->n_kv_heads), dim3(kSelThreads), smem, ctx->stream, *c, r->row_slot, r->row_pos, q,
                   (size_t)ldq, G, n_first, n_recent, n_select, chunk, sel);
    LAUNCH_CHECK(ctx);
    return B200_OK;
}
