// paged_attend.cu — one query row over a list of blocks of its context (b200_paged_attend).
//
//     x_j = cap(scale * q.k_j),  o = sum_j exp(x_j - max x) v_j / sum_j exp(x_j - max x)
// over the keys j <= position of the listed blocks. One pass with a running maximum and sum; a row without a key gives 0.
//
// One cluster of CTAs per (row, kv head) shares out the listed blocks; each CTA's four warps walk 16-key tiles of their own
// through private cp.async rings, and the warps' and the CTAs' states (accumulators, maximum, sum) are joined in shared
// memory, the CTAs' through distributed shared memory: nothing is parked in global memory, so the call needs no workspace
// and calls on several streams share nothing.
//
// Products run on mma.sync m16n8k16 over the fp16 cache with fp32 accumulation; f32 queries and weights are split into
// fp16 hi + lo parts (x = hi + lo to 2^-22), so the result keeps fp32 accuracy. S[head][key] = Q K^T takes the group's
// heads as rows; the context is accumulated transposed, O^T[dim][head] = V^T P^T, where a lane's scores are already the
// second operand. A tile's context starts from zero and is added to the running one by a rounded fma: the matrix unit cuts off
// what it adds to, and over the tiles of a long list that went one way (2048 keys: 1.5e-6 of the result, 3e-7 so). Rows of the last tile behind the position are filled with zeros by the copy: what the pool holds there
// (a NaN, say) meets a weight of 0 and must not be multiplied.
#include "paged.cuh"

namespace {

constexpr int kAttWarps = 4, kAttThreads = 32 * kAttWarps, kAttStages = 3;
constexpr int kAttMaxList = 2048;

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
__device__ __forceinline__ void split2(float x, float y, unsigned& hi, unsigned& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const unsigned*>(&h);
    lo = *reinterpret_cast<const unsigned*>(&l);
}

template <int HD>
struct AttendShape {
    static constexpr int KS = HD / 16, CPR = HD / 8, ROWB = HD * 2, TILE = 16 * ROWB, CPL = 16 * CPR / 32;
    static constexpr size_t ring = (size_t)kAttWarps * kAttStages * 2 * TILE;
};

template <int HD>
__global__ void __launch_bounds__(kAttThreads) paged_attend_kernel(const b200_paged_cache c, const int32_t* __restrict__ row_slot,
                                                                   const int32_t* __restrict__ row_pos, const float* __restrict__ q, size_t ldq, int G,
                                                                   float scale, float cap, const int32_t* __restrict__ sel, int n_select,
                                                                   float* __restrict__ out, size_t ldo) {
    using S = AttendShape<HD>;
    constexpr int KS = S::KS, CPR = S::CPR, ROWB = S::ROWB, TILE = S::TILE, CPL = S::CPL;
    extern __shared__ __align__(128) uint8_t att_smem[];  // rings, then the list: page and first key of each block
    int2* list = reinterpret_cast<int2*>(att_smem + S::ring);
    __shared__ int s_count[kAttWarps];
    const int ctas = (int)cluster_size(), rank = (int)cluster_rank();
    const int r = blockIdx.x / ctas, kvh = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
    const int slot = row_slot[r], pos = row_pos[r], br = c.block_rows;
    if (!paged_row_ok(slot, pos, c.n_seqs)) return;  // the whole cluster leaves; the row's output stays as it was

    // the listed blocks that hold a key the row sees, in the list's order
    const int have = paged_visible(pos, br, c.max_blocks);
    const int n_keys = min(pos, have * br - 1) + 1;
    const int32_t* tbl = c.block_table + (size_t)slot * c.max_blocks;
    const int32_t* lp = sel + ((size_t)r * c.n_kv_heads + kvh) * n_select;
    int n_list = 0;
    for (int i0 = 0; i0 < n_select; i0 += kAttThreads) {
        const int b = i0 + tid < n_select ? lp[i0 + tid] : -1;
        const int page = b >= 0 && b < have ? tbl[b] : 0;
        const bool in = paged_block_ok(page, c.n_blocks);
        const unsigned ballot = __ballot_sync(0xffffffffu, in);
        if (lane == 0) s_count[warp] = __popc(ballot);
        __syncthreads();
        int at = n_list + __popc(ballot & ((1u << lane) - 1u));
        for (int w = 0; w < kAttWarps; w++) {
            if (w < warp) at += s_count[w];
            n_list += s_count[w];
        }
        if (in) list[at] = make_int2(page, b * br);
        __syncthreads();
    }

    // the head's largest |q| is brought to [1, 2) by a power of two, which the scale gives back: neither a query beyond fp16's
    // range nor one among its subnormals loses anything
    unsigned qh0[KS], qh2[KS], ql0[KS], ql2[KS];
    {
        const float* qp = q + (size_t)r * ldq + (size_t)(kvh * G + (gid < G ? gid : 0)) * HD;
        float2 qa[KS], qb[KS];
        float most = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            qa[ks] = *reinterpret_cast<const float2*>(qp + 16 * ks + 2 * tig);
            qb[ks] = *reinterpret_cast<const float2*>(qp + 16 * ks + 8 + 2 * tig);
            most = fmaxf(fmaxf(most, fmaxf(fabsf(qa[ks].x), fabsf(qa[ks].y))), fmaxf(fabsf(qb[ks].x), fabsf(qb[ks].y)));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int e = (int)(__float_as_uint(most) >> 23) - 127;
        const int shift = most > 0.f && e < 128 ? max(-100, min(100, e)) : 0;
        const float down = gid < G ? __uint_as_float((unsigned)(127 - shift) << 23) : 0.f;
        scale *= __uint_as_float((unsigned)(127 + shift) << 23);
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            split2(qa[ks].x * down, qa[ks].y * down, qh0[ks], ql0[ks]);
            split2(qb[ks].x * down, qb[ks].y * down, qh2[ks], ql2[ks]);
        }
    }
    float o[KS][4];
#pragma unroll
    for (int mt = 0; mt < KS; mt++) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;

    // this warp's tiles: t0 + warp, t0 + warp + 4, ... of the cluster's n_list * (br / 16)
    const int tpb = br >> 4, tiles = n_list * tpb;
    const int t0 = (int)((long long)tiles * rank / ctas), t1 = (int)((long long)tiles * (rank + 1) / ctas);
    const int n_mine = t0 + warp < t1 ? (t1 - t0 - warp + kAttWarps - 1) / kAttWarps : 0;
    const unsigned ring = (unsigned)__cvta_generic_to_shared(att_smem) + (unsigned)(warp * kAttStages * 2 * TILE);
    auto first_key = [&](int it, int& page, int& row0) {
        const int t = t0 + warp + kAttWarps * it, e = t / tpb;
        row0 = (t - e * tpb) << 4;
        page = list[e].x;
        return list[e].y + row0;
    };
    auto issue = [&](int it) {
        if (it < n_mine) {
            int page, row0;
            const int key0 = first_key(it, page, row0);
            const size_t off = paged_tile(page, kvh, c.n_kv_heads, br, HD) + (size_t)row0 * HD;
            const uint8_t* ks = reinterpret_cast<const uint8_t*>(static_cast<const __half*>(c.k_pool) + off);
            const uint8_t* vs = reinterpret_cast<const uint8_t*>(static_cast<const __half*>(c.v_pool) + off);
            const unsigned dst = ring + (unsigned)((it % kAttStages) * 2 * TILE);
#pragma unroll
            for (int i = 0; i < CPL; i++) {
                const int ci = lane + 32 * i, row = ci / CPR, ch = ci % CPR;
                const unsigned d = (unsigned)(row * ROWB + ((ch ^ (row & 7)) << 4));
                const bool there = key0 + row < n_keys;
                copy16(dst + d, ks + ci * 16, there);
                copy16(dst + TILE + d, vs + ci * 16, there);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s < kAttStages - 1; s++) issue(s);

    const int lrow = (lane & 7) + ((lane >> 4) << 3), lsel = (lane >> 3) & 1;
    for (int it = 0; it < n_mine; it++) {
        issue(it + kAttStages - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(kAttStages - 1) : "memory");
        __syncwarp();
        const unsigned kb = ring + (unsigned)((it % kAttStages) * 2 * TILE), vb = kb + TILE;
        int page, row0;
        const int key0 = first_key(it, page, row0);
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
        float x[4] = {s0h[0] + s0l[0], s0h[1] + s0l[1], s1h[0] + s1l[0], s1h[1] + s1l[1]};
        const int kk[4] = {key0 + 2 * tig, key0 + 2 * tig + 1, key0 + 8 + 2 * tig, key0 + 9 + 2 * tig};
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[i] *= scale;  // this lane's scores are all of head gid
            if (cap != 0.f) x[i] = cap * tanhf(x[i] / cap);
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
            p[i] = __expf(x[i] - m_ref);
            ps += p[i];
        }
        ps += __shfl_xor_sync(0xffffffffu, ps, 1);
        ps += __shfl_xor_sync(0xffffffffu, ps, 2);
        l_run = l_run * alpha + ps;
        m_run = m_new;
        unsigned ph0, pl0, ph1, pl1;
        split2(p[0], p[1], ph0, pl0);
        split2(p[2], p[3], ph1, pl1);
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
        __syncwarp();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    // join the warps (in the rings' room): acc[warp][head][dim], then maximum and sum [warp][head]; the CTA's own state
    // lies behind them, where the cluster reads it
    float* acc = reinterpret_cast<float*>(att_smem);
    float* sm_m = acc + kAttWarps * G * HD;
    float* sm_l = sm_m + kAttWarps * G;
    float* cta = sm_l + kAttWarps * G;  // [G][HD], [G] maximum, [G] sum
    if (tig == 0 && gid < G) {
        sm_m[warp * G + gid] = m_run;
        sm_l[warp * G + gid] = l_run;
    }
#pragma unroll
    for (int mt = 0; mt < KS; mt++) {
        const int h0 = 2 * tig, h1 = h0 + 1, d0 = 16 * mt + gid;
        if (h0 < G) { acc[(warp * G + h0) * HD + d0] = o[mt][0]; acc[(warp * G + h0) * HD + d0 + 8] = o[mt][2]; }
        if (h1 < G) { acc[(warp * G + h1) * HD + d0] = o[mt][1]; acc[(warp * G + h1) * HD + d0 + 8] = o[mt][3]; }
    }
    __syncthreads();
    for (int idx = tid; idx < G * HD; idx += kAttThreads) {
        const int g = idx / HD, e = idx % HD;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kAttWarps; w++) M = fmaxf(M, sm_m[w * G + g]);
        const float ref = M == -INFINITY ? 0.f : M;
        float tot = 0.f, l = 0.f;
#pragma unroll
        for (int w = 0; w < kAttWarps; w++) {
            const float f = __expf(sm_m[w * G + g] - ref);
            tot += acc[(w * G + g) * HD + e] * f;
            l += sm_l[w * G + g] * f;
        }
        cta[idx] = tot;
        if (e == 0) {
            cta[G * HD + g] = M;
            cta[G * HD + G + g] = l;
        }
    }
    cluster_sync();
    // every CTA joins its share of the outputs over all CTAs, in their order
    for (int idx = rank * kAttThreads + tid; idx < G * HD; idx += ctas * kAttThreads) {
        const int g = idx / HD;
        float M = -INFINITY;
        for (int w = 0; w < ctas; w++) M = fmaxf(M, cluster_load_f32(cluster_addr(cta + G * HD + g, w)));
        const float ref = M == -INFINITY ? 0.f : M;
        float tot = 0.f, l = 0.f;
        for (int w = 0; w < ctas; w++) {
            const float f = __expf(cluster_load_f32(cluster_addr(cta + G * HD + g, w)) - ref);
            tot += cluster_load_f32(cluster_addr(cta + idx, w)) * f;
            l += cluster_load_f32(cluster_addr(cta + G * HD + G + g, w)) * f;
        }
        out[(size_t)r * ldo + (size_t)kvh * G * HD + idx] = l > 0.f || l != l ? tot / l : 0.f;
    }
    cluster_sync();  // no CTA leaves while another reads its state
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
    if (!(scale >= 0.f) || !(softcap >= 0.f) || scale > 3.4e38f || softcap > 3.4e38f)
        B200_FAIL(ctx, B200_BAD_ARGUMENT, "b200_paged_attend: scale %g and softcap %g must be finite and not negative", (double)scale, (double)softcap);
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
    const int G = n_heads / c->n_kv_heads, tiles = n_select * (c->block_rows / 16);
    const float s = scale != 0.f ? scale : 1.0f / sqrtf((float)c->head_dim);
    int ctas = 1;
    while (ctas < 8 && (long long)r->n_rows * c->n_kv_heads * ctas < 4 * ctx->sm_count && tiles / ctas > 8) ctas *= 2;
    const dim3 grid((unsigned)(r->n_rows * ctas), c->n_kv_heads);
    static SmemLimit limit[2];
    if (c->head_dim == 128) {
        CUDA_TRY(ctx, limit[1].raise(paged_attend_kernel<128>, ctx->device, AttendShape<128>::ring + sizeof(int2) * kAttMaxList));
        launch_cluster(paged_attend_kernel<128>, ctas, grid, dim3(kAttThreads), AttendShape<128>::ring + sizeof(int2) * n_select, ctx->stream, *c, r->row_slot,
                       r->row_pos, q, (size_t)ldq, G, s, softcap, sel, n_select, out, (size_t)ldo);
    } else {
        CUDA_TRY(ctx, limit[0].raise(paged_attend_kernel<64>, ctx->device, AttendShape<64>::ring + sizeof(int2) * kAttMaxList));
        launch_cluster(paged_attend_kernel<64>, ctas, grid, dim3(kAttThreads), AttendShape<64>::ring + sizeof(int2) * n_select, ctx->stream, *c, r->row_slot,
                       r->row_pos, q, (size_t)ldq, G, s, softcap, sel, n_select, out, (size_t)ldo);
    }
    LAUNCH_CHECK(ctx);
    return B200_OK;
}
