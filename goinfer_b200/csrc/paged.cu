// paged.cu — a paged KV cache in the caller's own device memory: the block tables, free stack, packed rows and slot map
// of a step from its request lengths (b200_paged_plan), and the store of a step's K/V rows with the bounds of their keys
// (b200_paged_append).
//
// plan. Sequence i keeps len_i rows and takes new_i more, in blocks of br rows:
//     want_i = ceil((len_i + new_i) / br),  grow_i = max(0, want_i - have_i),  shrink_i = max(0, have_i - want_i)
// With G = sum grow and S = sum shrink, element e of the released blocks (sequence, then table position, ascending) is
// pushed as number S-1-e, and element k of the new blocks is popped as number k: what the k-th new block pops is
// stack[count + S - 1 - k], which for k < S is the k-th released block. Three scans (rows, grow, shrink) over the sequences
// place everything; each released block, new block and row then finds its sequence by a search in the scan.
// The scans are latency (a chain of loads, a scan, loads), so one CTA makes them; with many blocks to move it is a cluster, whose
// CTAs each make the scans for themselves and share the blocks out. Barriers stand between the reads of the old state, the
// pushes and the pops. Up to 2048 rows are written by the same launch, more by a second kernel over the whole GPU.
#include "paged.cuh"

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanMaxSeqs = 16384;  // three scans of 4 bytes a sequence in shared memory

struct PlanArgs {
    int32_t* table;
    int32_t* seq_blocks;
    int32_t* stack;
    int32_t* count;
    const int32_t* kv_len;
    const int32_t* n_new;
    int32_t *row0, *row_slot, *row_pos, *slot_map, *status;
    int n_seqs, n_blocks, max_blocks, block_rows, n_rows;
    unsigned by_rows;  // division by block_rows: paged_divisor
    int top_step;      // the first step of a search among n_seqs
};

// the last index i with scan[i] <= e, for e < scan[n] (empty sequences are stepped over)
__device__ __forceinline__ int find_owner(const int* scan, int n, int top_step, int e) {
    int at = 0;
    for (int step = top_step; step > 0; step >>= 1)
        if (at + step < n && scan[at + step] <= e) at += step;
    return at;
}

// the packed row r, whose sequence is i and starts at row `first`
__device__ __forceinline__ void write_row(const PlanArgs& a, int r, int i, int first, int len) {
    const int pos = len + r - first, p = (int)paged_div((unsigned)pos, a.by_rows);
    const int block = __ldcg(a.table + (size_t)i * a.max_blocks + p);
    a.row_slot[r] = i;
    a.row_pos[r] = pos;
    a.slot_map[r] = paged_block_ok(block, a.n_blocks) ? block * a.block_rows + (pos - p * a.block_rows) : -1;
}

struct Sums {
    long long rows;
    int grow, shrink;
};

__device__ __forceinline__ Sums warp_inclusive(Sums v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long r = __shfl_up_sync(0xffffffffu, v.rows, o);
        const int g = __shfl_up_sync(0xffffffffu, v.grow, o), s = __shfl_up_sync(0xffffffffu, v.shrink, o);
        if (lane >= o) { v.rows += r; v.grow += g; v.shrink += s; }
    }
    return v;
}

__global__ void __launch_bounds__(kPlanThreads, 1) paged_plan_kernel(const PlanArgs a, int write_rows) {
    pdl_trigger();
    pdl_wait();
    extern __shared__ int plan_smem[];
    int* row0 = plan_smem;                    // [n + 1] scan of new rows
    int* grow0 = row0 + a.n_seqs + 1;         // [n + 1] scan of blocks taken
    int* shrink0 = grow0 + a.n_seqs + 1;      // [n + 1] scan of blocks given back
    __shared__ Sums warp_sum[32];
    __shared__ int first_bad;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, n = a.n_seqs, br = a.block_rows;
    if (tid == 0) first_bad = n;
    __syncthreads();

    // every thread takes a run of sequences; with more than one it looks at them again for the scan
    const int per = (n + threads - 1) / threads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    const int free0 = *a.count;
    int add = 0, want = 0, have = 0;
    auto look = [&](int i) {
        const int len = a.kv_len[i];
        add = a.n_new[i];
        have = a.seq_blocks[i];
        const long long all = (long long)len + add;
        const bool bad = len < 0 || add < 0 || all > (long long)a.max_blocks * br || have < 0 || have > a.max_blocks || len > (long long)have * br;
        if (bad) atomicMin(&first_bad, i);
        want = bad ? have : (int)paged_div_up((unsigned)all, a.by_rows);
        if (bad) add = 0;
    };
    Sums mine{0, 0, 0};
    for (int i = i0; i < i1; i++) {
        look(i);
        mine.rows += add;
        mine.grow += max(0, want - have);
        mine.shrink += max(0, have - want);
    }
    Sums scan = warp_inclusive(mine, lane);
    if (lane == 31) warp_sum[warp] = scan;
    __syncthreads();
    if (warp == 0) {
        const Sums t = warp_inclusive(32 * lane < threads ? warp_sum[lane] : Sums{0, 0, 0}, lane);
        warp_sum[lane] = t;
    }
    __syncthreads();
    const Sums total = warp_sum[31];
    scan.rows -= mine.rows;
    scan.grow -= mine.grow;
    scan.shrink -= mine.shrink;
    if (warp > 0) {
        scan.rows += warp_sum[warp - 1].rows;
        scan.grow += warp_sum[warp - 1].grow;
        scan.shrink += warp_sum[warp - 1].shrink;
    }
    for (int i = i0; i < i1; i++) {
        if (per > 1) look(i);
        row0[i] = (int)scan.rows;  // used only when the rows fit n_rows
        grow0[i] = scan.grow;
        shrink0[i] = scan.shrink;
        scan.rows += add;
        scan.grow += max(0, want - have);
        scan.shrink += max(0, have - want);
    }
    const int G = total.grow, S = total.shrink;
    if (tid == 0) {
        row0[n] = (int)total.rows;
        grow0[n] = G;
        shrink0[n] = S;
    }
    const int bad_seq = first_bad;
    const bool bad = bad_seq < n || total.rows > a.n_rows || free0 < 0 || (long long)free0 + S > a.n_blocks;
    const bool full = !bad && G > free0 + S;
    const int rank = (int)cluster_rank(), ctas = (int)cluster_size();
    const int gtid = rank * threads + tid, step = ctas * threads;
    auto everyone = [&] {
        if (ctas > 1) cluster_sync(); else __syncthreads();
    };
    everyone();  // the old state has been read by every CTA

    if (gtid == 0) {
        a.status[0] = bad ? B200_BAD_ARGUMENT : full ? B200_KV_POOL_FULL : B200_OK;
        a.status[1] = bad || full ? 0 : (int)total.rows;
        a.status[2] = bad || full ? free0 : free0 + S - G;
        a.status[3] = bad ? bad_seq : full ? G - free0 - S : 0;
        if (!bad && !full) *a.count = free0 + S - G;
    }
    const bool go = !bad && !full;  // else nothing changes, and no row takes part in what follows
    for (int i = gtid; i <= n; i += step) a.row0[i] = go ? row0[i] : 0;
    if (go) {
        auto want_of = [&](int i) { return (int)paged_div_up((unsigned)a.kv_len[i] + (unsigned)a.n_new[i], a.by_rows); };
        for (int i = gtid; i < n; i += step) a.seq_blocks[i] = want_of(i);
        for (int e = gtid; e < S; e += step) {
            const int i = find_owner(shrink0, n, a.top_step, e);
            int32_t* entry = a.table + (size_t)i * a.max_blocks + want_of(i) + (e - shrink0[i]);
            a.stack[free0 + S - 1 - e] = *entry;
            *entry = 0;
        }
        if (S > 0) everyone();  // the pushes are on the stack
        for (int e = gtid; e < G; e += step) {
            const int i = find_owner(grow0, n, a.top_step, e);  // its new blocks end at want_of(i)
            a.table[(size_t)i * a.max_blocks + want_of(i) + (e - grow0[i + 1])] = __ldcg(a.stack + free0 + S - 1 - e);
        }
    }
    if (write_rows) {
        if (go && G > 0) everyone();  // the table is written
        const int rows = go ? (int)total.rows : 0;
        for (int r = gtid; r < a.n_rows; r += step) {
            if (r < rows) {
                const int i = find_owner(row0, n, a.top_step, r);
                write_row(a, r, i, row0[i], a.kv_len[i]);
            } else {
                a.row_slot[r] = a.row_pos[r] = a.slot_map[r] = -1;
            }
        }
    }
}

constexpr int kRowThreads = 256;

// A row a thread; the sequences' first rows are searched in shared memory.
__global__ void __launch_bounds__(kRowThreads) paged_rows_kernel(const PlanArgs a) {
    extern __shared__ int plan_smem[];
    pdl_trigger();
    pdl_wait();
    const int n = a.n_seqs;
    for (int i = threadIdx.x; i <= n; i += kRowThreads) plan_smem[i] = __ldcg(a.row0 + i);
    __syncthreads();
    const int rows = plan_smem[n];  // 0 when the plan did not go through
    for (int r = blockIdx.x * kRowThreads + threadIdx.x; r < a.n_rows; r += gridDim.x * kRowThreads) {
        if (r < rows) {
            const int i = find_owner(plan_smem, n, a.top_step, r);
            write_row(a, r, i, plan_smem[i], a.kv_len[i]);
        } else {
            a.row_slot[r] = a.row_pos[r] = a.slot_map[r] = -1;
        }
    }
}

// ---- append ----------------------------------------------------------------------------------------------------------
// Packed rows whose slots follow one another inside one block are a run; the CTA that holds a run's first row stores the whole
// run, so a block's bounds are written once and see every key: lo_d = min, hi_d = max over the block's rows 0 .. last of the
// fp16 keys, the older ones read back from the pool. NaN keys make NaN bounds (min.NaN / max.NaN).
//
// Bytes bound it: 8 HD in and 4 HD out a row and head. A warp takes a kv head of the run (four dims a lane, one row of 128 or two
// of 64 at a time) with four loads of k and of v in flight (with eight, at twice the
// registers, 8192-row prompts run alike and decode rows 0.2 us slower); where there are fewer heads than warps, several warps share a
// head's rows and join their bounds in shared memory.
constexpr int kAppendMaxWarps = 16;

struct Bounds4 {  // of four dims
    uint2 lo = {0x7c007c00u, 0x7c007c00u}, hi = {0xfc00fc00u, 0xfc00fc00u};  // +inf, -inf
    __device__ __forceinline__ void fold(uint2 l, uint2 h) {
        lo.x = min_nan2(lo.x, l.x); lo.y = min_nan2(lo.y, l.y);
        hi.x = max_nan2(hi.x, h.x); hi.y = max_nan2(hi.y, h.y);
    }
};
__device__ __forceinline__ uint2 to_half4(float4 x) {
    const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
    return make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}

// rows_per_cta: packed rows whose runs a CTA looks for; parts: warps that share a head (when above 1, the CTA has heads * parts warps)
template <int HD>
__global__ void __launch_bounds__(32 * kAppendMaxWarps) paged_append_kernel(const b200_paged_cache c, const int32_t* slot_map, int n_rows,
                                                                            const float* k, size_t ldk, const float* v,
                                                                            size_t ldv, int rows_per_cta, int parts) {
    pdl_trigger();
    pdl_wait();
    constexpr int LPR = HD / 4, RPW = 32 / LPR, U = 4, OLD = 16;  // lanes a row, rows a warp at a time, loads in flight of new and of older rows
    __shared__ Bounds4 joined[kAppendMaxWarps][LPR];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, br = c.block_rows;
    const int sub = lane % LPR, row_of = lane / LPR;
    // the first rows of runs among this CTA's rows, a lane a row
    const int mine = blockIdx.x * rows_per_cta + lane;
    bool starts = false;
    if (lane < rows_per_cta && mine < n_rows) {
        const int at = slot_map[mine], before = mine > 0 ? slot_map[mine - 1] : -1;
        starts = at >= 0 && paged_block_ok(at / br, c.n_blocks) && (before != at - 1 || at % br == 0);
    }
    for (unsigned todo = __ballot_sync(0xffffffffu, starts); todo; todo &= todo - 1u) {
        const int r = blockIdx.x * rows_per_cta + __ffs((int)todo) - 1, at = slot_map[r], block = at / br, first = at % br;
        const int most = min(br - first, n_rows - r);
        int n = 0;
        while (n < most) {
            const unsigned here = __ballot_sync(0xffffffffu, n + lane < most && slot_map[r + n + lane] == at + n + lane);
            n += here == 0xffffffffu ? 32 : __ffs((int)~here) - 1;
            if (here != 0xffffffffu) break;
        }
        for (int u = warp; u < c.n_kv_heads * parts; u += warps) {
            const int h = u % c.n_kv_heads, part = u / c.n_kv_heads;
            const size_t tile = paged_tile(block, h, c.n_kv_heads, br, HD);
            uint2* kt = reinterpret_cast<uint2*>(static_cast<__half*>(c.k_pool) + tile) + sub;
            uint2* vt = reinterpret_cast<uint2*>(static_cast<__half*>(c.v_pool) + tile) + sub;
            const float4* ks = reinterpret_cast<const float4*>(k + (size_t)r * ldk + (size_t)h * HD) + sub;
            const float4* vs = reinterpret_cast<const float4*>(v + (size_t)r * ldv + (size_t)h * HD) + sub;
            Bounds4 bounds;
            const int j0 = n * part / parts, j1 = n * (part + 1) / parts;
            for (int j = j0 + row_of; j < j1; j += U * RPW) {
                float4 kx[U], vx[U];
#pragma unroll
                for (int i = 0; i < U; i++) {
                    if (j + i * RPW < j1) {
                        kx[i] = __ldcs(ks + (size_t)(j + i * RPW) * (ldk / 4));
                        vx[i] = __ldcs(vs + (size_t)(j + i * RPW) * (ldv / 4));
                    }
                }
#pragma unroll
                for (int i = 0; i < U; i++) {
                    if (j + i * RPW < j1) {
                        const uint2 ko = to_half4(kx[i]);
                        const size_t to = (size_t)(first + j + i * RPW) * LPR;
                        kt[to] = ko;
                        vt[to] = to_half4(vx[i]);
                        bounds.fold(ko, ko);
                    }
                }
            }
            if (!c.key_bounds) continue;
            const int o0 = first * part / parts, o1 = first * (part + 1) / parts;
            for (int j = o0 + row_of; j < o1; j += OLD * RPW) {
                uint2 old[OLD];
#pragma unroll
                for (int i = 0; i < OLD; i++)
                    if (j + i * RPW < o1) old[i] = kt[(size_t)(j + i * RPW) * LPR];
#pragma unroll
                for (int i = 0; i < OLD; i++)
                    if (j + i * RPW < o1) bounds.fold(old[i], old[i]);
            }
            if constexpr (RPW == 2) {
                const uint2 l = make_uint2(__shfl_xor_sync(0xffffffffu, bounds.lo.x, 16), __shfl_xor_sync(0xffffffffu, bounds.lo.y, 16));
                const uint2 g = make_uint2(__shfl_xor_sync(0xffffffffu, bounds.hi.x, 16), __shfl_xor_sync(0xffffffffu, bounds.hi.y, 16));
                bounds.fold(l, g);
            }
            if (parts > 1) {
                if (row_of == 0) joined[warp][sub] = bounds;
                __syncthreads();
                if (part == 0)
                    for (int p = 1; p < parts; p++) bounds.fold(joined[warp + p * c.n_kv_heads][sub].lo, joined[warp + p * c.n_kv_heads][sub].hi);
                __syncthreads();
            }
            if (part == 0 && row_of == 0) {
                uint2* b = reinterpret_cast<uint2*>(static_cast<__half*>(c.key_bounds) + ((size_t)block * c.n_kv_heads + h) * 2 * HD) + sub;
                b[0] = bounds.lo;
                b[LPR] = bounds.hi;
            }
        }
    }
}

}  // namespace

int paged_check(b200_ctx* ctx, const char* what, const b200_paged_cache* c, const b200_paged_rows* r, PagedNeeds need) {
    if (!c || !r) B200_FAIL(ctx, B200_BAD_ARGUMENT, "%s: null cache or rows", what);
    if (c->n_seqs < 1 || c->max_blocks < 1 || c->n_blocks < 2 || c->block_rows < 16 || c->block_rows > 256 || c->block_rows % 16 != 0)
        B200_FAIL(ctx, B200_BAD_ARGUMENT,
                  "%s: %d sequences of %d table entries over %d blocks of %d rows; a cache has at least one sequence and entry, two blocks "
                  "(block 0 is the null block) and blocks of 16 to 256 rows, a multiple of 16", what, c->n_seqs, c->max_blocks, c->n_blocks, c->block_rows);
    if ((long long)c->n_blocks * c->block_rows > 0x7fffffffLL || (long long)c->max_blocks * c->block_rows > 0x7fffffffLL)
        B200_FAIL(ctx, B200_BAD_ARGUMENT, "%s: a pool and a table hold fewer than 2^31 rows each", what);
    if (!c->block_table || paged_misaligned(c->block_table, 4)) B200_FAIL(ctx, B200_BAD_ARGUMENT, "%s: block_table is null or not 4-byte aligned", what);
    if (r->n_rows < 0 || r->n_rows > 1 << 27) B200_FAIL(ctx, B200_BAD_ARGUMENT, "%s: %d rows; at most 2^27", what, r->n_rows);
    if (r->n_rows > 0 && (need.stack || !need.map) && (!r->row_slot || !r->row_pos || paged_misaligned(r->row_slot, 4) || paged_misaligned(r->row_pos, 4)))
        B200_FAIL(ctx, B200_BAD_ARGUMENT, "%s: row_slot or row_pos is null or not 4-byte aligned", what);
    if (need.map && r->n_rows > 0 && (!r->slot_map || paged_misaligned(r->slot_map, 4)))
        B200_FAIL(ctx, B200_BAD_ARGUMENT, "%s: slot_map is null or not 4-byte aligned", what);
    if (need.stack) {
        if (!c->seq_blocks || !c->free_blocks || !c->free_count || !r->seq_row0 || !r->status || paged_misaligned(c->seq_blocks, 4) ||
            paged_misaligned(c->free_blocks, 4) || paged_misaligned(c->free_count, 4) || paged_misaligned(r->seq_row0, 4) || paged_misaligned(r->status, 4))
            B200_FAIL(ctx, B200_BAD_ARGUMENT, "%s: seq_blocks, free_blocks, free_count, seq_row0 or status is null or not 4-byte aligned", what);
    }
    if (need.pools || need.bounds) {
        if (c->n_kv_heads < 1 || !(c->head_dim == 64 || c->head_dim == 128))
            B200_FAIL(ctx, B200_BAD_ARGUMENT, "%s: %d kv heads of %d; head_dim is 64 or 128", what, c->n_kv_heads, c->head_dim);
        if (need.pools && (!c->k_pool || !c->v_pool || paged_misaligned(c->k_pool, 16) || paged_misaligned(c->v_pool, 16)))
            B200_FAIL(ctx, B200_BAD_ARGUMENT, "%s: a pool is null or not 16-byte aligned", what);
        if (need.bounds ? (!c->key_bounds || paged_misaligned(c->key_bounds, 16)) : paged_misaligned(c->key_bounds, 16))
            B200_FAIL(ctx, B200_BAD_ARGUMENT, "%s: key_bounds is null or not 16-byte aligned", what);
    }
    return B200_OK;
}

extern "C" int b200_paged_plan(b200_ctx* ctx, const b200_paged_cache* c, const b200_paged_rows* r, const int32_t* kv_len, const int32_t* n_new) {
    if (!ctx) return B200_BAD_ARGUMENT;
    PagedNeeds need;
    need.stack = need.map = true;
    ST_TRY(paged_check(ctx, "b200_paged_plan", c, r, need));
    if (!kv_len || !n_new || paged_misaligned(kv_len, 4) || paged_misaligned(n_new, 4))
        B200_FAIL(ctx, B200_BAD_ARGUMENT, "b200_paged_plan: kv_len or n_new is null or not 4-byte aligned");
    if (c->n_seqs > kPlanMaxSeqs || (long long)c->n_seqs * c->max_blocks > 0x7fffffffLL)
        B200_FAIL(ctx, B200_BAD_ARGUMENT, "b200_paged_plan: %d sequences of %d table entries; at most %d sequences and 2^31 - 1 entries in all", c->n_seqs,
                  c->max_blocks, kPlanMaxSeqs);
    if (ctx->device < 0) B200_FAIL(ctx, B200_CUDA_ERROR, "b200_paged_plan: the context has no device");
    DeviceScope dev;
    CUDA_TRY(ctx, dev.enter(ctx->device));
    int top_step = 1;
    while (top_step * 2 < c->n_seqs) top_step *= 2;
    const PlanArgs a{c->block_table, c->seq_blocks, c->free_blocks, c->free_count, kv_len, n_new, r->seq_row0, r->row_slot, r->row_pos, r->slot_map,
                     r->status, c->n_seqs, c->n_blocks, c->max_blocks, c->block_rows, r->n_rows, paged_divisor(c->block_rows), top_step};
    static SmemLimit limit, rows_limit;
    const size_t scan = sizeof(int) * ((size_t)c->n_seqs + 1);
    CUDA_TRY(ctx, limit.raise(paged_plan_kernel, ctx->device, 3 * sizeof(int) * (kPlanMaxSeqs + 1)));
    const bool apart = r->n_rows > 2 * kPlanThreads;
    // Sequences and blocks enough for four a thread: a cluster. Two calls with a cluster and with one CTA, in us, sequences x rows: 2000 x
    // 32 16.5 and 21.4, 1000 x 60 14.0 and 17.9, 5000 x 8 22.8 and 27.4, 5000 x 1 21.1 and 21.9, 4000 x 1 19.4 and 18.9; below the
    // border 2000 x 1 13.9 and 13.5, 64 x 1 8.9 and 7.0, 1000 x 30 14.2 either way, but 256 x 200 12.0 and 14.6.
    const int ctas = c->n_seqs + r->n_rows / c->block_rows > 4 * kPlanThreads ? 8 : 1;
    // A decode step's lengths do with eight warps, whose barriers are the cheaper. Two calls with 8 and with 32 warps: 1 sequence of 1 row 5.6
    // and 6.4 us, 64 x 1 6.1 and 7.0, 256 x 1 7.0 and 7.6, 64 x 8 7.1 and 7.2; behind the border 256 x 2 8.0 and 7.7, 300 x 1 9.0 and
    // 7.9, 1000 x 1 13.1 and 9.6.
    const int threads = c->n_seqs <= 256 && r->n_rows <= 512 ? 256 : kPlanThreads;
    launch_cluster(paged_plan_kernel, ctas, dim3(ctas), dim3(threads), 3 * scan, ctx->stream, a, apart ? 0 : 1);
    if (apart) {
        LAUNCH_CHECK(ctx);
        CUDA_TRY(ctx, rows_limit.raise(paged_rows_kernel, ctx->device, sizeof(int) * (kPlanMaxSeqs + 1)));
        const int most = 2 * ctx->sm_count, blocks = ceil_div(r->n_rows, kRowThreads);
        launch_pdl(paged_rows_kernel, dim3(blocks < most ? blocks : most), dim3(kRowThreads), scan, ctx->stream, a);
    }
    LAUNCH_CHECK(ctx);
    return B200_OK;
}

extern "C" int b200_paged_append(b200_ctx* ctx, const b200_paged_cache* c, const b200_paged_rows* r, const float* k, int ldk, const float* v, int ldv) {
    if (!ctx) return B200_BAD_ARGUMENT;
    PagedNeeds need;
    need.pools = need.map = true;
    ST_TRY(paged_check(ctx, "b200_paged_append", c, r, need));
    if (r->n_rows == 0) return B200_OK;
    const long long width = (long long)c->n_kv_heads * c->head_dim;
    if (!k || !v || paged_misaligned(k, 16) || paged_misaligned(v, 16) || ldk < width || ldv < width || (ldk & 3) || (ldv & 3))
        B200_FAIL(ctx, B200_BAD_ARGUMENT,
                  "b200_paged_append: k and v must be 16-byte aligned with strides of at least %lld floats, a multiple of 4 (got %d and %d)", width, ldk, ldv);
    if (ctx->device < 0) B200_FAIL(ctx, B200_CUDA_ERROR, "b200_paged_append: the context has no device");
    DeviceScope dev;
    CUDA_TRY(ctx, dev.enter(ctx->device));
    // Few rows are decode steps: a CTA looks at one, and while there is an SM for each, with tall blocks sixteen warps share the
    // older rows to be read. With sixteen and with eight warps, 64 decode rows of 8 heads of 128 in blocks of 16, 32, 64, 256: 3.5 and 3.4,
    // 3.8 and 4.1, 4.4 and 5.1, 8.7 and 12.6 us; of 4 heads of 64 in blocks of 32, 64, 128, 256: 3.4 and 3.3, 3.6 and 3.5, 3.9 and
    // 4.1, 4.6 and 5.2; 200 rows of 8 heads of 128 in blocks of 64, 256: 7.3 and 5.8, 22.5 and 27.7. (What decides is how many CTAs hold a
    // run, which the rows alone do not say: seven chunks of 301 rows of 8 heads of 128 would take 12.9 us with sixteen, 17.4 with eight, in
    // blocks of 64; of 4 heads of 64 in blocks of 32 5.9 and 4.9.)
    // Many rows are prompts, whose runs fill blocks: a CTA that finds no run among its rows costs about as much as 4 ns of the GPU, so it
    // looks at more, as long as four CTAs an SM are left (32768 rows of 8 heads of 128 in blocks of 64: 139, 82, 74, 68 us with 1, 4, 8, 32
    // rows a CTA; 2115 rows in seven chunks with blocks of 32: 8.1, 5.3, 5.5, 7.2 us; 5529 rows of one head of 64 in 291 chunks: 6.9 us
    // with 16, 8.4 with 32).
    int rows = 1;
    while (rows < 32 && r->n_rows > 4 * ctx->sm_count * rows) rows *= 2;
    const int warps = r->n_rows <= ctx->sm_count && c->block_rows >= 32 ? kAppendMaxWarps : 8;
    const int parts = c->n_kv_heads < warps ? warps / c->n_kv_heads : 1;
    const int threads = 32 * (c->n_kv_heads < warps ? c->n_kv_heads * parts : warps);
    auto kernel = c->head_dim == 128 ? paged_append_kernel<128> : paged_append_kernel<64>;
    launch_cluster(kernel, 1, dim3(ceil_div(r->n_rows, rows)), dim3(threads), 0, ctx->stream, *c, r->slot_map, r->n_rows, k, (size_t)ldk, v, (size_t)ldv, rows,
                   parts);
    LAUNCH_CHECK(ctx);
    return B200_OK;
}
