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
// split leaves at most 2^-22 |q_d| or 2^-36; a step that adds 16 products to the sum is off by at most 17 * 2^-23 of the terms'
// absolute sum S, 16 of them by 2^-14.9 S. E = 2^-13 S + 2^-12 covers it (128 dims of the largest fp16 bound times 2^-36 are
// 2^-13), with S from the absolute values of the same operands. The true m-th score lies within E of the m-th s~, so a block whose s~ is more than
// 2E above (below) that is in (out) for certain; only the blocks between (a handful) are scored in f64. An infinity or a
// NaN anywhere makes E infinite, and every block is scored in f64.
//
// One cluster of CTAs per (row, kv head): the CTAs share out the blocks and send s~ to the first CTA's shared memory, which
// selects: a histogram of the scores' range in 2048 bins finds the bin of the m-th (and is taken again inside the bin
// while that is wider than E), and one ordered pass writes the list.
#include "paged.cuh"

namespace {

constexpr int kSelThreads = 128, kSelWarps = kSelThreads / 32;
constexpr int kSelMaxBlocks = 24576;  // 8 bytes a block in the first CTA's shared memory
constexpr int kSelMaxList = 2048;
constexpr int kSelBins = 2048;
constexpr int kSelDoubt = 256;        // blocks in doubt that are ranked in a list; more are selected among in place
constexpr int kSelMaxCluster = 8;
constexpr unsigned long long kSelIn = ~0ull, kSelOut = 0ull;  // no score has these keys

__device__ __forceinline__ void mma16816(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// f over the values of all threads; two barriers, and one more before `red` may be used again
template <typename T, typename F>
__device__ __forceinline__ T block_fold(T v, T* red, F f) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    T t = red[0];
#pragma unroll
    for (int w = 1; w < kSelWarps; w++) t = f(t, red[w]);
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
#pragma unroll
    for (int w = 0; w < kSelWarps; w++) {
        if (w < warp) before += red[w];
        total += red[w];
    }
    return before + s - v;
}

// The thread's bins (top first) hold `hist`; finds the bin in which the running count from the top reaches `need`.
__device__ __forceinline__ void find_bin(const unsigned* hist, int need, int* red, int* s_bin, int* s_above, int* s_in) {
    constexpr int BPT = kSelBins / kSelThreads;
    const int first = kSelBins - 1 - (int)threadIdx.x * BPT;
    int mine = 0;
#pragma unroll
    for (int j = 0; j < BPT; j++) mine += (int)hist[first - j];
    int total;
    int above = block_scan(mine, red, total);
    if (above < need && above + mine >= need) {
        for (int j = 0; j < BPT; j++) {
            const int here = (int)hist[first - j];
            if (above + here >= need) {
                *s_bin = first - j;
                *s_above = above;
                *s_in = here;
                break;
            }
            above += here;
        }
    }
    __syncthreads();
}

// f64 score of one block by the HD/8 lanes that share it (eight dims each, `sub` among them); every lane gets it. The
// bounds' order of summation is the same for every block, so equal bounds have equal scores.
template <int HD>
__device__ __forceinline__ double exact_score(const b200_paged_cache& c, int page, int kvh, const float* q, int G, int sub) {
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
    for (int g = 0; g < G; g++) {
        double s = 0.0;
#pragma unroll
        for (int d = 0; d < 8; d++) {
            const float x = q[(size_t)g * HD + 8 * sub + d];
            s = fma((double)x, (double)__half2float(x > 0.f ? hh[d] : lh[d]), s);
        }
#pragma unroll
        for (int o = LPB / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        nan |= s != s;
        best = fmax(best, s);
    }
    best = nan ? top : fmin(fmax(best, -top), top) + 0.0;  // -0 -> +0
    return ok ? best : -top;
}

template <int HD>
__global__ void __launch_bounds__(kSelThreads) paged_select_kernel(const b200_paged_cache c, const int32_t* __restrict__ row_slot,
                                                                   const int32_t* __restrict__ row_pos, const float* __restrict__ q, size_t ldq, int G,
                                                                   int n_first, int n_recent, int n_select, int32_t* __restrict__ sel) {
    // first CTA, per middle block: s~ (low word) until the blocks are told apart, then kSelIn, kSelOut or an f64 key
    extern __shared__ __align__(16) unsigned long long sel_slot[];
    __shared__ unsigned hist[kSelBins];
    __shared__ float s_err[kSelMaxCluster * kSelWarps];
    __shared__ float red_f[kSelWarps];
    __shared__ int red_i[kSelWarps];
    __shared__ unsigned long long red_u[kSelWarps], doubt_key[kSelDoubt];
    __shared__ int doubt[kSelDoubt];
    __shared__ int s_bin, s_above, s_in, s_doubt;
    const int ctas = (int)cluster_size(), rank = (int)cluster_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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
    const float* qr = q + (size_t)r * ldq + (size_t)kvh * G * HD;
    cluster_sync();  // the first CTA has started: its shared memory may be written
    if (m > 0) {
        // Fragments: row of A = block, column of B = head. A lane's words of a 16-byte chunk are taken as the dims of its
        // places in the k steps; q is laid out by the same rule, so a bound is loaded as it lies.
        constexpr int CH = HD / 32;  // 16-byte chunks of a row per lane: chunks tig, tig + 4, ...
        const int gid = lane >> 2, tig = lane & 3;
        unsigned ph[CH][4], nh[CH][4], pl[CH][4], nl[CH][4];  // q > 0 and q <= 0, parts hi and lo; word j: dims 2j, 2j + 1
        float f0, f1;  // the columns' powers of two against the group's largest
        {
            const float* qp = qr + (size_t)(gid < G ? gid : 0) * HD + 8 * tig;
            float4 x[CH][2];
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < CH; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    x[i][h] = *reinterpret_cast<const float4*>(qp + 32 * i + 4 * h);
                    most = fmaxf(fmaxf(most, fmaxf(fabsf(x[i][h].x), fabsf(x[i][h].y))), fmaxf(fabsf(x[i][h].z), fabsf(x[i][h].w)));
                }
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            // the head's largest |q| comes to [1, 2); 2^-126 and less count as 2^-126 (the floor of E covers them)
            const int e = max(-126, min(127, (int)(__float_as_uint(most) >> 23) - 127));
            const float down0 = pow2(-(e / 2)), down1 = pow2(-(e - e / 2));  // 2^-e in two factors, each of them normal
            int e_max = gid < G && most > 0.f ? e : -126;
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) e_max = max(e_max, __shfl_xor_sync(0xffffffffu, e_max, o));
            const float f = gid < G ? pow2(max(-126, e - e_max)) : 0.f;
            f0 = __shfl_sync(0xffffffffu, f, 8 * tig);
            f1 = __shfl_sync(0xffffffffu, f, 8 * tig + 4);
            auto split = [](float a, float b, unsigned& hi, unsigned& lo) {
                hi = half2_bits(a, b);
                const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                lo = half2_bits((a - t.x) * 2048.f, (b - t.y) * 2048.f);
            };
#pragma unroll
            for (int i = 0; i < CH; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float4 v = x[i][j >> 1];
                    const float a = ((j & 1) ? v.z : v.x) * down0 * down1, b = ((j & 1) ? v.w : v.y) * down0 * down1;
                    // !(q > 0) goes with the lower bounds, a NaN as well
                    split(a > 0.f ? a : 0.f, b > 0.f ? b : 0.f, ph[i][j], pl[i][j]);
                    split(a > 0.f ? 0.f : a, b > 0.f ? 0.f : b, nh[i][j], nl[i][j]);
                }
        }
        const unsigned slots0 = cluster_addr(sel_slot, 0);
        float err = 0.f;
        const int step = 16 * kSelWarps * ctas;
        int b0 = 16 * (rank * kSelWarps + warp);
        auto page_of = [&](int b) { return b < n ? tbl[b] : 0; };
        int page0 = page_of(b0 + gid), page1 = page_of(b0 + 8 + gid);
        for (; b0 < n; b0 += step) {
            const bool ok0 = paged_block_ok(page0, c.n_blocks), ok1 = paged_block_ok(page1, c.n_blocks);
            const size_t head = (size_t)c.n_kv_heads, bytes = 4 * HD;
            const uint8_t* p0 = static_cast<const uint8_t*>(c.key_bounds) + ((size_t)(ok0 ? page0 : 0) * head + kvh) * bytes + 16 * tig;
            const uint8_t* p1 = static_cast<const uint8_t*>(c.key_bounds) + ((size_t)(ok1 ? page1 : 0) * head + kvh) * bytes + 16 * tig;
            uint4 l0[CH], l1[CH], h0[CH], h1[CH];
#pragma unroll
            for (int i = 0; i < CH; i++) {
                const uint4 z = make_uint4(0, 0, 0, 0);
                l0[i] = ok0 ? __ldg(reinterpret_cast<const uint4*>(p0 + 64 * i)) : z;
                h0[i] = ok0 ? __ldg(reinterpret_cast<const uint4*>(p0 + 2 * HD + 64 * i)) : z;
                l1[i] = ok1 ? __ldg(reinterpret_cast<const uint4*>(p1 + 64 * i)) : z;
                h1[i] = ok1 ? __ldg(reinterpret_cast<const uint4*>(p1 + 2 * HD + 64 * i)) : z;
            }
            page0 = page_of(b0 + step + gid);
            page1 = page_of(b0 + step + 8 + gid);
            float hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0}, up[4] = {0, 0, 0, 0}, dn[4] = {0, 0, 0, 0};
            auto two = [&](const uint4& a, const uint4& b, int i, int j, bool upper) {  // words j and j + 1 of a chunk: one k step
                const unsigned a0 = j ? a.z : a.x, a1 = j ? b.z : b.x, a2 = j ? a.w : a.y, a3 = j ? b.w : b.y;
                constexpr unsigned abs2 = 0x7fff7fffu;
                if (upper) {
                    mma16816(hi, a0, a1, a2, a3, ph[i][j], ph[i][j + 1]);
                    mma16816(lo, a0, a1, a2, a3, pl[i][j], pl[i][j + 1]);
                    mma16816(up, a0 & abs2, a1 & abs2, a2 & abs2, a3 & abs2, ph[i][j], ph[i][j + 1]);
                } else {
                    mma16816(hi, a0, a1, a2, a3, nh[i][j], nh[i][j + 1]);
                    mma16816(lo, a0, a1, a2, a3, nl[i][j], nl[i][j + 1]);
                    mma16816(dn, a0 & abs2, a1 & abs2, a2 & abs2, a3 & abs2, nh[i][j], nh[i][j + 1]);
                }
            };
#pragma unroll
            for (int i = 0; i < CH; i++) {
                two(h0[i], h1[i], i, 0, true);
                two(l0[i], l1[i], i, 0, false);
                two(h0[i], h1[i], i, 2, true);
                two(l0[i], l1[i], i, 2, false);
            }
            // columns 2 tig and 2 tig + 1 of rows gid (values 0, 1) and gid + 8 (values 2, 3)
            float s[2], E[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float S0 = up[2 * h] - dn[2 * h], S1 = up[2 * h + 1] - dn[2 * h + 1];
                const float s0 = fmaf(lo[2 * h], 0x1p-11f, hi[2 * h]) * f0, s1 = fmaf(lo[2 * h + 1], 0x1p-11f, hi[2 * h + 1]) * f1;
                const float E0 = fmaf(S0, 0x1p-13f, 0x1p-12f) * f0, E1 = fmaf(S1, 0x1p-13f, 0x1p-12f) * f1;
                const bool in0 = 2 * tig < G, in1 = 2 * tig + 1 < G;
                s[h] = fmaxf(in0 ? s0 : -INFINITY, in1 ? s1 : -INFINITY);
                E[h] = fmaxf(in0 ? E0 : 0.f, in1 ? E1 : 0.f);
                // an infinity or a NaN shows in S (0 * inf) or in s
                if ((in0 && !(fabsf(E0) + fabsf(s0) < 3e38f)) || (in1 && !(fabsf(E1) + fabsf(s1) < 3e38f))) E[h] = INFINITY;
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) {
                    s[h] = fmaxf(s[h], __shfl_xor_sync(0xffffffffu, s[h], o));
                    E[h] = fmaxf(E[h], __shfl_xor_sync(0xffffffffu, E[h], o));
                }
            }
            if (ok0) err = fmaxf(err, E[0]);
            if (ok1) err = fmaxf(err, E[1]);
            if (tig == 0 && b0 + gid < n) cluster_store_u64(slots0 + 8u * (unsigned)(b0 + gid), __float_as_uint(ok0 ? s[0] : -INFINITY));
            if (tig == 0 && b0 + 8 + gid < n) cluster_store_u64(slots0 + 8u * (unsigned)(b0 + 8 + gid), __float_as_uint(ok1 ? s[1] : -INFINITY));
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) err = fmaxf(err, __shfl_xor_sync(0xffffffffu, err, o));
        if (lane == 0) cluster_store_f32(cluster_addr(s_err + rank * kSelWarps + warp, 0), err);
    }
    cluster_sync();  // the scores are in the first CTA's shared memory
    if (rank != 0) return;

    for (int i = tid; i < n_first; i += kSelThreads) out[i] = i;
    for (int i = tid; i < n_recent; i += kSelThreads) out[n_select - n_recent + i] = have - n_recent + i;
    if (m <= 0) return;
    float err = 0.f;
    for (int i = 0; i < ctas * kSelWarps; i++) err = fmaxf(err, s_err[i]);
    err *= 1.01f;  // what the comparisons below round
    auto approx = [&](int i) { return __uint_as_float((unsigned)sel_slot[i]); };
    auto least = [](float a, float b) { return fminf(a, b); };
    auto most = [](float a, float b) { return fmaxf(a, b); };

    // [lo, hi]: holds the m-th largest s~. Unmapped blocks count as the least s~: too much, but never enough to be in for certain.
    float lo = -INFINITY, hi = INFINITY, floor_s = 0.f;
    if (err < INFINITY) {
        float mn = INFINITY, mx = -INFINITY;
        for (int i = tid; i < n; i += kSelThreads) {
            const float s = approx(i);
            if (s > -INFINITY) { mn = fminf(mn, s); mx = fmaxf(mx, s); }
        }
        lo = block_fold(mn, red_f, least);
        hi = block_fold(mx, red_f, most);
        if (!(lo <= hi)) lo = hi = 0.f;  // nothing is mapped
        floor_s = lo;
        int need = m;
        for (int pass = 0; pass < 3 && hi - lo > err; pass++) {
            const float inv = (float)(kSelBins - 1) / (hi - lo);
            for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kSelThreads) {
                const float s = fmaxf(approx(i), floor_s);
                if (s >= lo && s <= hi) atomicAdd(&hist[min(kSelBins - 1, (int)((s - lo) * inv))], 1u);
            }
            __syncthreads();
            find_bin(hist, need, red_i, &s_bin, &s_above, &s_in);
            const int bin = s_bin, above = s_above, here = s_in;
            mn = INFINITY;
            mx = -INFINITY;
            for (int i = tid; i < n; i += kSelThreads) {
                const float s = fmaxf(approx(i), floor_s);
                if (s >= lo && s <= hi && min(kSelBins - 1, (int)((s - lo) * inv)) == bin) { mn = fminf(mn, s); mx = fmaxf(mx, s); }
            }
            lo = block_fold(mn, red_f, least);
            hi = block_fold(mx, red_f, most);
            need -= above;
            if (need == here) hi = lo;       // the m-th is the bin's least
            else if (need == 1) lo = hi;     // ... or its largest
        }
    }
    // in for certain, out for certain, in doubt
    const float sure_in = hi + 2.f * err, sure_out = lo - 2.f * err;
    if (tid == 0) s_doubt = 0;
    __syncthreads();
    int in = 0;
    for (int i = tid; i < n; i += kSelThreads) {
        const float s = fmaxf(approx(i), floor_s);
        if (s > sure_in) {
            in++;
            sel_slot[i] = kSelIn;
        } else if (s < sure_out) {
            sel_slot[i] = kSelOut;
        } else {
            const int at = atomicAdd(&s_doubt, 1);
            if (at < kSelDoubt) doubt[at] = i;
            sel_slot[i] = 1;  // in doubt: no f64 score has this key
        }
    }
    in = block_fold(in, red_i, [](int a, int b) { return a + b; });
    const int n_doubt = s_doubt;
    int need = m - in;  // 1 .. n_doubt of those in doubt
    unsigned long long kmin = kSelIn, kmax = kSelIn;  // the list: keys above kmax, and the first `need` from kmin to kmax
    constexpr int LPB = HD / 8, BPW = 32 / LPB;
    const int sub = lane % LPB, part = lane / LPB;
    if (n_doubt == need) {
        kmin = 1;
        need = m;
    } else if (n_doubt <= kSelDoubt) {
        for (int j0 = warp * BPW; j0 < n_doubt; j0 += kSelWarps * BPW) {
            const int j = j0 + part;
            const double s = exact_score<HD>(c, j < n_doubt ? tbl[doubt[j]] : 0, kvh, qr, G, sub);
            if (sub == 0 && j < n_doubt) doubt_key[j] = key_of(s);
        }
        __syncthreads();
        for (int j = tid; j < n_doubt; j += kSelThreads) {
            const unsigned long long k = doubt_key[j];
            const int i = doubt[j];
            int before = 0;
            for (int t = 0; t < n_doubt; t++) before += doubt_key[t] > k || (doubt_key[t] == k && doubt[t] < i);
            sel_slot[i] = before < need ? kSelIn : kSelOut;
        }
        need = m;
    } else {
        __syncthreads();
        for (int i0 = warp * BPW; i0 < n; i0 += kSelWarps * BPW) {
            const int i = i0 + part;
            const bool here = i < n && sel_slot[i] == 1;
            if (!__any_sync(0xffffffffu, here)) continue;
            const double s = exact_score<HD>(c, here ? tbl[i] : 0, kvh, qr, G, sub);
            __syncwarp();
            if (sub == 0 && here) sel_slot[i] = key_of(s);
        }
        __syncthreads();
        kmin = kSelIn;
        kmax = kSelOut;
        for (int i = tid; i < n; i += kSelThreads) {
            const unsigned long long k = sel_slot[i];
            if (k != kSelIn && k != kSelOut) {
                kmin = min(kmin, k);
                kmax = max(kmax, k);
            }
        }
        kmin = block_fold(kmin, red_u, [](unsigned long long a, unsigned long long b) { return a < b ? a : b; });
        kmax = block_fold(kmax, red_u, [](unsigned long long a, unsigned long long b) { return a < b ? b : a; });
        while (true) {  // at most six divisions of a 64-bit range by 2048
            const int width = 64 - __clzll((long long)(kmax - kmin));
            const int shift = width > 11 ? width - 11 : 0;
            __syncthreads();
            for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kSelThreads) {
                const unsigned long long k = sel_slot[i];
                if (k >= kmin && k <= kmax) atomicAdd(&hist[(unsigned)((k - kmin) >> shift)], 1u);
            }
            __syncthreads();
            find_bin(hist, need, red_i, &s_bin, &s_above, &s_in);
            need -= s_above;
            const unsigned long long from = kmin + ((unsigned long long)s_bin << shift), to = from + ((1ull << shift) - 1ull);
            kmax = to < kmax ? to : kmax;
            kmin = from;
            if (s_in == need || shift == 0) break;
        }
    }
    __syncthreads();
    // an ordered pass over runs of blocks: a run a thread
    const int per = (n + kSelThreads - 1) / kSelThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    int n_above = 0, n_edge = 0;
    for (int i = i0; i < i1; i++) {
        n_above += sel_slot[i] > kmax;
        n_edge += sel_slot[i] >= kmin && sel_slot[i] <= kmax;
    }
    int total;
    const int above0 = block_scan(n_above, red_i, total);
    int edge = block_scan(n_edge, red_i, total);
    int at = n_first + above0 + min(edge, need);
    for (int i = i0; i < i1; i++) {
        const unsigned long long k = sel_slot[i];
        const bool is_edge = k >= kmin && k <= kmax;
        if (k > kmax || (is_edge && edge < need)) out[at++] = n_first + i;
        edge += is_edge;
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
    auto kernel = c->head_dim == 128 ? paged_select_kernel<128> : paged_select_kernel<64>;
    static SmemLimit limit[2];
    const size_t smem = 8 * (size_t)c->max_blocks;
    CUDA_TRY(ctx, limit[c->head_dim == 128].raise(kernel, ctx->device, 8 * (size_t)kSelMaxBlocks));
    int ctas = 1;
    while (ctas < 8 && (long long)r->n_rows * c->n_kv_heads * ctas < 2 * ctx->sm_count && c->max_blocks / ctas > 64) ctas *= 2;
    launch_cluster(kernel, ctas, dim3((unsigned)(r->n_rows * ctas), c->n_kv_heads), dim3(kSelThreads), smem, ctx->stream, *c, r->row_slot, r->row_pos, q,
                   (size_t)ldq, G, n_first, n_recent, n_select, sel);
    LAUNCH_CHECK(ctx);
    return B200_OK;
}
