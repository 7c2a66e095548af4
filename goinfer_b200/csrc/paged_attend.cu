// paged_attend.cu — one query row over a list of blocks of its context (b200_paged_attend).
//
//     x_j = cap(scale * q.k_j),  o = sum_j exp(x_j - max x) v_j / sum_j exp(x_j - max x)
// over the keys j <= position of the listed blocks. One pass with a running maximum and sum; a row without a key gives 0.
//
// One cluster of CTAs per (row, kv head) shares out the listed blocks; each CTA's four warps walk 16-key tiles of their own
// through private cp.async rings, and the warps' states (accumulators, maximum, sum) are joined in shared memory. Each CTA of
// the cluster owns a share of the outputs: the others store their states of it into the owner's shared memory, and behind one
// cluster barrier the owner joins them. Nothing is parked in global memory, so the call needs no workspace and calls on
// several streams share nothing.
//
// Products run on mma.sync m16n8k16 over the fp16 cache with fp32 accumulation; f32 queries and weights are split into
// fp16 hi + lo parts. S[head][key] = Q K^T takes the group's heads as rows, the lo parts 2^11 times as large and in a sum of their
// own: with the head's largest |q| in [1, 2), a query keeps its 2^-22 down to 2^-14 and 2^-36 below, so that a small one still
// counts against a key of thousands; the context is accumulated transposed, O^T[dim][head] = V^T P^T, where a lane's scores are already the
// second operand. A tile's context starts from zero and is added to the running one by a rounded fma: the matrix unit cuts off
// what it adds to, and over the tiles of a long list that went one way (2048 keys: 1.5e-6 of the result, 4e-7 so). Rows of the
// last tile behind the position are filled with zeros by the copy: what the pool holds there (a NaN, say) meets a weight of 0
// and must not be multiplied.
//
// Weights. hi + lo is x to 2^-22 where the step of fp16's subnormals, 2^-24, is no more than 2^-21 of x: for x >= 2^-3. A weight is
// taken in 2^-15ths, p = 2^15 exp(x - m) <= 32768, in the context and in the sum alike, so this holds for those down to 2^-18 of the
// largest one that the warp has seen. Where a tile has a score 12.4 or more below the largest (a key far above the rest, say, whose
// own value may be next to nothing), what the halves left of the weights below 2^-3 is multiplied by V once more, 2^36 times as large, until
// none is below: every weight keeps its 2^-22 down to the smallest numbers of fp32. Measured against no care at all: the look costs up to
// 1 % (256 rows of 128 blocks 312.5 -> 313.2 us, 45 ragged rows 12.0 -> 12.3); where every tile has such a score 317 and 14.1 us.
#include "paged.cuh"

namespace {

constexpr int kAttWarps = 4, kAttThreads = 32 * kAttWarps, kAttStages = 2;
constexpr int kAttMaxList = 2048;
constexpr float kWeight = 0x1p15f, kSmall = 0x1p-3f, kStep = 0x1p36f, kFar = -12.4f;  // of the weights, see above; 2^-18 = exp(-12.48)
constexpr int kAttMaxCluster = 8;

__device__ __forceinline__ void ldm4(unsigned addr, unsigned (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldm4_t(unsigned addr, unsigned (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 bytes, or zeros when `there` is false (the source is then not read)
__device__ __forceinline__ void copy16(unsigned dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
// x and y as fp16 hi + lo / up
__device__ __forceinline__ void split2(float x, float y, unsigned& hi, unsigned& lo, float up = 1.f) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn((x - f.x) * up, (y - f.y) * up);
    hi = *reinterpret_cast<const unsigned*>(&h);
    lo = *reinterpret_cast<const unsigned*>(&l);
}

// A part's weight in the whole: f over the sum l; 0 where no key was seen, NaN where l is.
__device__ __forceinline__ float whole(float f, float l) { return l > 0.f || l != l ? f / l : 0.f; }

template <int HD>
struct AttendShape {
    static constexpr int KS = HD / 16, CPR = HD / 8, ROWB = HD * 2, TILE = 16 * ROWB, CPL = 16 * CPR / 32;
    static constexpr size_t ring = (size_t)kAttWarps * kAttStages * 2 * TILE;
    static constexpr size_t inbox = 8 * HD + 32 * (kAttMaxCluster - 1);  // what the CTAs send this one: of each, this one's share
    static constexpr size_t smem(int n_select) { return ring + sizeof(float) * inbox + sizeof(int2) * (size_t)n_select; }
    static constexpr int ACC = HD + 4;  // floats between heads in the warps' states: the fragments' stores meet no bank twice
};

// Two CTAs an SM at least: with all the registers that leaves it the compiler keeps more of a tile's steps in flight than it would
// by itself (4 x 131k keys 45.6 against 49.7 us; 256 rows 312 against 310). Four at head_dim 64: 128 registers, where the compiler takes
// 135 by itself and three fit (32/4 heads, 128 rows of 64 blocks 25.2 against 33.1 us, 256 rows 47.1 against 54.3; 200 rows, which then
// happen to fill the last wave, 44.2 against 38.7).
template <int HD>
__global__ void __launch_bounds__(kAttThreads, HD == 64 ? 4 : 2) paged_attend_kernel(const b200_paged_cache c, const int32_t* row_slot,
                                                                   const int32_t* row_pos, const float* q, size_t ldq, int G,
                                                                   float scale, float cap, const int32_t* sel, int n_select,
                                                                   float* out, size_t ldo) {
    pdl_wait();
    using S = AttendShape<HD>;
    constexpr int KS = S::KS, CPR = S::CPR, ROWB = S::ROWB, TILE = S::TILE, CPL = S::CPL;
    extern __shared__ __align__(128) uint8_t att_smem[];  // rings, inbox, then the list: page and first key of each block
    float* inbox = reinterpret_cast<float*>(att_smem + S::ring);
    int2* list = reinterpret_cast<int2*>(inbox + S::inbox);
    __shared__ int s_count[kAttWarps];
    __shared__ float s_max[kAttWarps][8], s_sum[kAttWarps][8], s_factor[kAttMaxCluster][8];  // [][head]
    __shared__ float in_max[kAttMaxCluster][8], in_sum[kAttMaxCluster][8];                   // of the cluster's CTAs
    const int ctas = (int)cluster_size(), rank = (int)cluster_rank();
    const int r = blockIdx.x / ctas, kvh = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
    // the row's place, the first entries of its list and its queries are fetched together
    const int32_t* lp = sel + ((size_t)r * c.n_kv_heads + kvh) * n_select;
    const int slot = row_slot[r], pos = row_pos[r], br = c.block_rows;
    int entry = tid < n_select ? lp[tid] : -1;
    float2 qa[KS], qb[KS];
    {
        const float* qp = q + (size_t)r * ldq + (size_t)(kvh * G + (gid < G ? gid : 0)) * HD;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            qa[ks] = *reinterpret_cast<const float2*>(qp + 16 * ks + 2 * tig);
            qb[ks] = *reinterpret_cast<const float2*>(qp + 16 * ks + 8 + 2 * tig);
        }
    }
    if (!paged_row_ok(slot, pos, c.n_seqs)) return;  // the whole cluster leaves; the row's output stays as it was
    if (ctas > 1) cluster_arrive();

    // the listed blocks that hold a key the row sees, in the list's order
    const int have = paged_visible(pos, br, c.max_blocks);
    const int n_keys = min(pos, have * br - 1) + 1;
    const int32_t* tbl = c.block_table + (size_t)slot * c.max_blocks;
    int n_list = 0;
    for (int i0 = 0; i0 < n_select; i0 += kAttThreads) {
        const int b = entry;
        if (i0 + kAttThreads < n_select) entry = i0 + kAttThreads + tid < n_select ? lp[i0 + kAttThreads + tid] : -1;
        const int page = b >= 0 && b < have ? tbl[b] : 0;
        const bool in = paged_block_ok(page, c.n_blocks);
        const unsigned ballot = __ballot_sync(0xffffffffu, in);
        if (i0 > 0) __syncthreads();  // the counts of the round before have been read
        if (lane == 0) s_count[warp] = __popc(ballot);
        __syncthreads();
        int at = n_list + __popc(ballot & ((1u << lane) - 1u));
#pragma unroll
        for (int w = 0; w < kAttWarps; w++) {
            if (w < warp) at += s_count[w];
            n_list += s_count[w];
        }
        if (in) list[at] = make_int2(page, b * br);
    }
    __syncthreads();

    // this warp's tiles: t0 + warp, t0 + warp + 4, ... of the cluster's n_list * (br / 16); (e, sub): block and tile in it
    const int tpb = br >> 4, tiles = n_list * tpb;
    const int t0 = tiles * rank / ctas, t1 = tiles * (rank + 1) / ctas;
    const int n_mine = t0 + warp < t1 ? (t1 - t0 - warp + kAttWarps - 1) / kAttWarps : 0;
    const unsigned ring = (unsigned)__cvta_generic_to_shared(att_smem) + (unsigned)(warp * kAttStages * 2 * TILE);
    const int de = kAttWarps / tpb, dsub = kAttWarps - de * tpb;
    struct Place {
        int e, sub;
    };
    auto advance = [&](Place& p) {
        p.e += de;
        p.sub += dsub;
        if (p.sub >= tpb) { p.sub -= tpb; p.e++; }
    };
    Place next{(t0 + warp) / tpb, 0};
    next.sub = t0 + warp - next.e * tpb;
    Place now = next;
    const size_t copy_at = (size_t)kvh * br * HD * 2 + 16 * lane;  // of a lane's first 16 bytes in a block
    const size_t block_bytes = (size_t)c.n_kv_heads * br * HD * 2;
    auto issue = [&](int it) {
        if (it < n_mine) {
            const int2 b = list[next.e];
            const int keys = n_keys - (b.y + 16 * next.sub);  // of the tile's sixteen, the ones that the row sees
            const size_t off = (size_t)b.x * block_bytes + copy_at + (size_t)(next.sub * TILE);
            const uint8_t *ks = static_cast<const uint8_t*>(c.k_pool) + off, *vs = static_cast<const uint8_t*>(c.v_pool) + off;
            const unsigned dst = ring + (unsigned)((it % kAttStages) * 2 * TILE);
#pragma unroll
            for (int i = 0; i < CPL; i++) {
                const int ci = lane + 32 * i, row = ci / CPR, ch = ci % CPR;
                const unsigned d = (unsigned)(row * ROWB + ((ch ^ (row & 7)) << 4));
                copy16(dst + d, ks + i * 512, row < keys);
                copy16(dst + TILE + d, vs + i * 512, row < keys);
            }
            advance(next);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s < kAttStages - 1; s++) issue(s);

    // the head's largest |q| is brought to [1, 2) by a power of two, which the scale gives back: queries may lie beyond fp16's range
    // or among its subnormals
    unsigned qh0[KS], qh2[KS], ql0[KS], ql2[KS];
    {
        float most = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
            most = fmaxf(fmaxf(most, fmaxf(fabsf(qa[ks].x), fabsf(qa[ks].y))), fmaxf(fabsf(qb[ks].x), fabsf(qb[ks].y)));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int e = (int)(__float_as_uint(most) >> 23) - 127;
        const int shift = most > 0.f && e < 128 ? max(-126, min(126, e)) : 0;
        const float down = gid < G ? __uint_as_float((unsigned)(127 - shift) << 23) : 0.f;
        scale *= __uint_as_float((unsigned)(127 + shift) << 23);
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            split2(qa[ks].x * down, qa[ks].y * down, qh0[ks], ql0[ks], 0x1p11f);
            split2(qb[ks].x * down, qb[ks].y * down, qh2[ks], ql2[ks], 0x1p11f);
        }
    }
    float o[KS][4];
#pragma unroll
    for (int mt = 0; mt < KS; mt++) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;

    const float inv_cap = cap != 0.f ? 1.f / cap : 0.f;
    const int lrow = (lane & 7) + ((lane >> 4) << 3), lsel = (lane >> 3) & 1;
    for (int it = 0; it < n_mine; it++) {
        issue(it + kAttStages - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(kAttStages - 1) : "memory");
        __syncwarp();
        const unsigned kb = ring + (unsigned)((it % kAttStages) * 2 * TILE), vb = kb + TILE;
        const int key0 = list[now.e].y + 16 * now.sub;
        advance(now);
        float s0h[4] = {0, 0, 0, 0}, s0l[4] = {0, 0, 0, 0}, s1h[4] = {0, 0, 0, 0}, s1l[4] = {0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            unsigned b[4];
            ldm4(kb + (unsigned)(lrow * ROWB + (((2 * ks + lsel) ^ (lrow & 7)) << 4)), b);
            mma16816(s0h, qh0[ks], 0u, qh2[ks], 0u, b[0], b[1]);
            mma16816(s1h, qh0[ks], 0u, qh2[ks], 0u, b[2], b[3]);
            mma16816(s0l, ql0[ks], 0u, ql2[ks], 0u, b[0], b[1]);
            mma16816(s1l, ql0[ks], 0u, ql2[ks], 0u, b[2], b[3]);
        }
        // (a score that is infinite says so in its upper part; the lower one, of any sign or zero times infinity, says nothing)
        auto joined = [](float hi, float lo) { return fabsf(hi) == INFINITY ? hi : fmaf(lo, 0x1p-11f, hi); };
        float x[4] = {joined(s0h[0], s0l[0]), joined(s0h[1], s0l[1]), joined(s1h[0], s1l[0]), joined(s1h[1], s1l[1])};
        const int kk[4] = {key0 + 2 * tig, key0 + 2 * tig + 1, key0 + 8 + 2 * tig, key0 + 9 + 2 * tig};
        float mx = -INFINITY, least = INFINITY;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[i] *= scale;  // this lane's scores are all of head gid
            if (cap != 0.f) x[i] = cap * tanhf(x[i] * inv_cap);
            least = fminf(least, x[i]);  // (of keys that the row does not see as well)
            if (kk[i] >= n_keys) x[i] = -INFINITY;
            mx = fmaxf(mx, x[i]);
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m_run, mx);
        const float m_ref = m_new == -INFINITY ? 0.f : m_new;  // nothing seen yet: every weight is exp(-inf) = 0
        const float alpha = __expf(m_run - m_ref);
        float p[4], ps = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            p[i] = kWeight * __expf(x[i] - m_ref);
            ps += p[i];
        }
        ps += __shfl_xor_sync(0xffffffffu, ps, 1);
        ps += __shfl_xor_sync(0xffffffffu, ps, 2);
        l_run = l_run * alpha + ps;
        m_run = m_new;
        unsigned ph0, pl0, ph1, pl1;
        split2(p[0], p[1], ph0, pl0);
        split2(p[2], p[3], ph1, pl1);
        const bool far = __any_sync(0xffffffffu, least - m_ref < kFar);  // a weight below kSmall, perhaps
        const float a0 = __shfl_sync(0xffffffffu, alpha, (2 * tig) * 4), a1 = __shfl_sync(0xffffffffu, alpha, (2 * tig + 1) * 4);
#pragma unroll
        for (int mt = 0; mt < KS; mt++) {
            unsigned v[4];
            ldm4_t(vb + (unsigned)(lrow * ROWB + (((2 * mt + lsel) ^ (lrow & 7)) << 4)), v);
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            mma16816(d, v[0], v[1], v[2], v[3], pl0, pl1);
            mma16816(d, v[0], v[1], v[2], v[3], ph0, ph1);
            o[mt][0] = fmaf(o[mt][0], a0, d[0]);
            o[mt][1] = fmaf(o[mt][1], a1, d[1]);
            o[mt][2] = fmaf(o[mt][2], a0, d[2]);
            o[mt][3] = fmaf(o[mt][3], a1, d[3]);
        }
        if (far) {
            bool more = true;  // at most four times: 2^-149 * 2^15 * 2^144 is above kSmall
            for (float down = 1.f / kStep; more; down *= 1.f / kStep) {
                auto left = [](float x, float y, unsigned hi, unsigned lo, float& a, float& b) {
                    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi)), l = __half22float2(*reinterpret_cast<const __half2*>(&lo));
                    a = fabsf(x) < kSmall ? ((x - h.x) - l.x) * kStep : 0.f;
                    b = fabsf(y) < kSmall ? ((y - h.y) - l.y) * kStep : 0.f;
                };
                left(p[0], p[1], ph0, pl0, p[0], p[1]);
                left(p[2], p[3], ph1, pl1, p[2], p[3]);
                more = false;
#pragma unroll
                for (int i = 0; i < 4; i++) more |= p[i] != 0.f && fabsf(p[i]) < kSmall;
                more = __any_sync(0xffffffffu, more);
                split2(p[0], p[1], ph0, pl0);
                split2(p[2], p[3], ph1, pl1);
#pragma unroll
                for (int mt = 0; mt < KS; mt++) {
                    unsigned v[4];
                    ldm4_t(vb + (unsigned)(lrow * ROWB + (((2 * mt + lsel) ^ (lrow & 7)) << 4)), v);
                    float d[4] = {0.f, 0.f, 0.f, 0.f};
                    mma16816(d, v[0], v[1], v[2], v[3], pl0, pl1);
                    mma16816(d, v[0], v[1], v[2], v[3], ph0, ph1);
#pragma unroll
                    for (int i = 0; i < 4; i++) o[mt][i] = fmaf(d[i], down, o[mt][i]);
                }
            }
        }
        __syncwarp();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    pdl_trigger();  // earlier gains nothing: lists that fill the GPU take the same time, few rows 0.1 to 0.2 us more
    __syncthreads();
    // join the warps (in the rings' room): acc[warp][head][dim]; maximum and sum [warp][head] become the warps' factors
    float* acc = reinterpret_cast<float*>(att_smem);
    if (tig == 0) {
        s_max[warp][gid] = m_run;
        s_sum[warp][gid] = l_run;
    }
#pragma unroll
    for (int mt = 0; mt < KS; mt++) {
        const int h0 = 2 * tig, h1 = h0 + 1, d0 = 16 * mt + gid;
        if (h0 < G) { acc[(warp * 8 + h0) * S::ACC + d0] = o[mt][0]; acc[(warp * 8 + h0) * S::ACC + d0 + 8] = o[mt][2]; }
        if (h1 < G) { acc[(warp * 8 + h1) * S::ACC + d0] = o[mt][1]; acc[(warp * 8 + h1) * S::ACC + d0 + 8] = o[mt][3]; }
    }
    if (ctas > 1) cluster_wait();  // the CTAs have started: their shared memory may be written
    __syncthreads();
    float M = -INFINITY, l = 0.f;
    if (warp == 0) {  // a lane: warp lane / 8, head gid of lane % 8
        const int w = lane >> 3, g = lane & 7;
#pragma unroll
        for (int i = 0; i < kAttWarps; i++) M = fmaxf(M, s_max[i][g]);
        const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int i = 0; i < kAttWarps; i++) l = fmaf(s_sum[i][g], __expf(s_max[i][g] - ref), l);
        const float f = __expf(s_max[w][g] - ref);
        s_factor[w][g] = ctas > 1 ? f : whole(f, l);
        for (int to = w; ctas > 1 && to < ctas; to += 4) {
            cluster_store(cluster_addr(&in_max[rank][g], to), M);
            cluster_store(cluster_addr(&in_sum[rank][g], to), l);
        }
    }
    __syncthreads();
    // Value idx of the CTA's state (head, dim) belongs to CTA (idx / 32) % ctas, where it is number idx / 32 / ctas * 32 + idx % 32:
    // what a warp sends goes to one CTA.
    const int values = G * HD, log_ctas = 31 - __clz(ctas), share = ((values >> 5) + ctas - 1) >> log_ctas << 5;
    float* out_row = out + (size_t)r * ldo + (size_t)kvh * values;
    for (int idx = tid; idx < values; idx += kAttThreads) {
        const int g = idx / HD, e = idx % HD;
        float tot = 0.f;
#pragma unroll
        for (int w = 0; w < kAttWarps; w++) tot = fmaf(acc[(w * 8 + g) * S::ACC + e], s_factor[w][g], tot);
        if (ctas == 1) out_row[idx] = tot;
        else cluster_store(cluster_addr(inbox + rank * share + ((idx >> (5 + log_ctas)) << 5 | (idx & 31)), (idx >> 5) & (ctas - 1)), tot);
    }
    if (ctas == 1) return;
    cluster_sync();  // what the CTAs sent has arrived
    if (tid < 8 * kAttMaxCluster) {
        const int w = tid >> 3, g = tid & 7;
        M = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < kAttMaxCluster; i++)
            if (i < ctas) M = fmaxf(M, in_max[i][g]);
        const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int i = 0; i < kAttMaxCluster; i++)
            if (i < ctas) l = fmaf(in_sum[i][g], __expf(in_max[i][g] - ref), l);
        if (w < ctas) s_factor[w][g] = whole(__expf(in_max[w][g] - ref), l);
    }
    __syncthreads();
    for (int i = tid; i < share; i += kAttThreads) {
        const int idx = ((i >> 5 << log_ctas) + rank) << 5 | (i & 31), g = idx / HD;
        if (idx >= values) break;
        float tot = 0.f;
#pragma unroll
        for (int w = 0; w < kAttMaxCluster; w++)
            if (w < ctas) tot = fmaf(inbox[w * share + i], s_factor[w][g], tot);
        out_row[idx] = tot;
    }
}

// As many CTAs a (row, kv head) as the GPU holds at once (two an SM at head_dim 128, four at 64), each with a tile a warp at
// least: one more wave costs more than the shorter share saves. Rows x kv heads x tiles, in us with 1, 2, 4, 8 CTAs:
// 8 x 64: 13.0, 9.4, 6.9, 5.9; 64 x 64: 13.4, 10.0, 8.5, 12.9; 128 x 64: 16.9, 16.5, 20.6, 29.9; 384 x 66: 45, 49, 60, 87.
// What the GPU holds is asked, not computed: 72 pairs at head_dim 128 (64 blocks of 16) take 13.4 us as clusters of 4 of which
// 71 fit, 9.6 as clusters of 2.
//
// At head_dim 64, with more than two CTAs an SM and no more than three, the launch asks for enough shared memory that a fourth
// does not fit. The clusters are otherwise placed four to an SM, which leaves a quarter of the SMs idle: 96 pairs x 64 tiles
// 8.8 -> 7.3 us, 192 pairs with lists of 48 to 66 tiles 12.8 -> 11.9; single CTAs, 440 pairs x 64, 22.1 -> 21.7. Below three an
// SM it is not worth it (32 pairs, 256 CTAs, 5.7 -> 5.9 with two an SM): the last clusters then no longer fit at once.
template <int HD>
int attend_launch(b200_ctx* ctx, const b200_paged_cache& c, const b200_paged_rows& r, const float* q, size_t ldq, int n_heads, float scale, float cap,
                  const int32_t* sel, int n_select, float* out, size_t ldo) {
    using S = AttendShape<HD>;
    constexpr size_t most = S::smem(kAttMaxList), three = 56 * 1024;  // of 228 KB an SM
    static_assert(HD == 128 || most < three, "");
    static SmemLimit limit;
    static ClusterFit fits, fits_three;
    auto kernel = paged_attend_kernel<HD>;
    CUDA_TRY(ctx, limit.raise(kernel, ctx->device, most > three ? most : three));
    const long long pairs = (long long)r.n_rows * c.n_kv_heads;
    const int tiles = n_select * (c.block_rows / 16);
    int lg = 0;
    for (int fit = 0; (kAttMaxCluster >> lg) > 1 && tiles >= (2 * kAttWarps) << lg; lg++) {
        CUDA_TRY(ctx, fits.count(kernel, ctx->device, lg + 1, dim3(kAttThreads), most, &fit));
        if (pairs > fit) break;
    }
    size_t smem = S::smem(n_select);
    if (HD == 64 && pairs << lg > 2ll * ctx->sm_count) {
        int fit = 0;
        CUDA_TRY(ctx, fits_three.count(kernel, ctx->device, lg, dim3(kAttThreads), three, &fit));
        if (pairs <= fit) smem = three;
    }
    launch_cluster(kernel, 1 << lg, dim3((unsigned)(r.n_rows << lg), c.n_kv_heads), dim3(kAttThreads), smem, ctx->stream, c, r.row_slot, r.row_pos, q, ldq,
                   n_heads / c.n_kv_heads, scale, cap, sel, n_select, out, ldo);
    LAUNCH_CHECK(ctx);
    return B200_OK;
}

}  // namespace

extern "C" int b200_paged_attend(b200_ctx* ctx, const b200_paged_cache* c, const b200_paged_rows* r, const float* q, int ldq, int n_heads, float scale,
                                 float softcap, const int32_t* sel, int n_select, float* out, int ldo) {
    if (!ctx) return B200_BAD_ARGUMENT;
    PagedNeeds need;
    need.pools = true;
    ST_TRY(paged_check(ctx, "b200_paged_attend", c, r, need));
    if (n_heads < 1 || n_heads % c->n_kv_heads || n_heads / c->n_kv_heads > 8)
        B200_FAIL(ctx, B200_BAD_ARGUMENT, "b200_paged_attend: %d query heads over %d kv heads; a group has 1 to 8 query heads", n_heads, c->n_kv_heads);
    if (n_select < 1 || n_select > kAttMaxList) B200_FAIL(ctx, B200_BAD_ARGUMENT, "b200_paged_attend: lists of %d blocks; 1 to %d", n_select, kAttMaxList);
    if (!(scale >= 0.f) || !(softcap >= 0.f) || scale > 3.4e38f || softcap > 3.4e38f || (softcap > 0.f && softcap < 1e-30f))
        B200_FAIL(ctx, B200_BAD_ARGUMENT, "b200_paged_attend: scale %g and softcap %g must be finite and not negative, a softcap 0 or at least 1e-30",
                  (double)scale, (double)softcap);
    if (r->n_rows == 0) return B200_OK;
    const long long width = (long long)n_heads * c->head_dim;
    if (!q || !sel || !out || paged_misaligned(q, 16) || paged_misaligned(sel, 4) || paged_misaligned(out, 16) || ldq < width || (ldq & 3) || ldo < width ||
        (ldo & 3))
        B200_FAIL(ctx, B200_BAD_ARGUMENT, "b200_paged_attend: q and out must be 16-byte aligned with strides of at least %lld floats, a multiple of 4 (got %d "
                                          "and %d); sel 4-byte aligned", width, ldq, ldo);
    if (c->n_kv_heads > 65535) B200_FAIL(ctx, B200_BAD_ARGUMENT, "b200_paged_attend: %d kv heads", c->n_kv_heads);
    if (ctx->device < 0) B200_FAIL(ctx, B200_CUDA_ERROR, "b200_paged_attend: the context has no device");
    DeviceScope dev;
    CUDA_TRY(ctx, dev.enter(ctx->device));
    const float s = scale != 0.f ? scale : 1.0f / sqrtf((float)c->head_dim);
    if (c->head_dim == 128) return attend_launch<128>(ctx, *c, *r, q, (size_t)ldq, n_heads, s, softcap, sel, n_select, out, (size_t)ldo);
    return attend_launch<64>(ctx, *c, *r, q, (size_t)ldq, n_heads, s, softcap, sel, n_select, out, (size_t)ldo);
}
