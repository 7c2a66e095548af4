// paged.cuh — what the operators over a caller-owned paged cache (paged.cu, paged_select.cu, paged_attend.cu) share:
// address rules that hold on the host and on the device, cluster primitives, the checks of the host structs.
#pragma once
#include <atomic>

#include "common.cuh"

// A table entry names a block of the pools when it lies in 1 .. n_blocks-1 (block 0 is the null block). Every kernel asks
// this before it forms an address, so a table that holds anything else reads and writes nothing.
__host__ __device__ inline bool paged_block_ok(int block, int n_blocks) { return block > 0 && block < n_blocks; }

// A packed row takes part when it names a sequence and a position; the rows behind the last sequence are marked -1.
__host__ __device__ inline bool paged_row_ok(int slot, int pos, int n_seqs) { return slot >= 0 && slot < n_seqs && pos >= 0; }

// Table positions that a row at `pos` sees (a position past the table sees the whole table).
__host__ __device__ inline int paged_visible(int pos, int block_rows, int max_blocks) {
    const int b = pos / block_rows;
    return (b < max_blocks ? b : max_blocks - 1) + 1;
}

// Division by block_rows (16 d, d <= 16) of x < 2^31 without the instruction sequence of a division: x / 16d = (x >> 4) / d,
// and y / d = y * ceil(2^31 / d) >> 31 for y < 2^27, because y times what the ceiling adds (below 1) stays below 2^31 / d.
inline unsigned paged_divisor(int block_rows) { return (unsigned)(((1ull << 31) + (unsigned)block_rows / 16 - 1) / ((unsigned)block_rows / 16)); }
__host__ __device__ inline unsigned paged_div(unsigned x, unsigned divisor) { return (unsigned)(((unsigned long long)(x >> 4) * divisor) >> 31); }
__host__ __device__ inline unsigned paged_div_up(unsigned x, unsigned divisor) { return x == 0 ? 0 : paged_div(x - 1, divisor) + 1; }

// Halves in front of row 0 of a block's tile of one kv head. 64-bit: a pool passes 2^31 elements at 4 GB.
__host__ __device__ inline size_t paged_tile(int block, int kvh, int n_kv, int block_rows, int hd) {
    return ((size_t)block * n_kv + kvh) * block_rows * hd;
}

// Checks of the structs that every entry point makes (paged.cu). need_*: which arrays the call touches.
struct PagedNeeds {
    bool pools = false, bounds = false, stack = false, map = false;
};
int paged_check(b200_ctx*, const char* what, const b200_paged_cache*, const b200_paged_rows*, PagedNeeds);

inline bool paged_misaligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

// Raises a kernel's dynamic shared memory limit once per device. Two contexts of one device may come here at the same
// time: the flag is set after the attribute, which may be set twice.
struct SmemLimit {
    std::atomic<bool> done[64] = {};
    template <typename K>
    cudaError_t raise(K* kernel, int device, size_t bytes) {
        if (device < 0 || device >= 64) return cudaErrorInvalidDevice;
        if (done[device].load(std::memory_order_acquire)) return cudaSuccess;
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e == cudaSuccess) done[device].store(true, std::memory_order_release);
        return e;
    }
};

#ifdef __CUDACC__
// How many clusters of 2^lg CTAs of a kernel the GPU holds at once, asked once per device. A cluster stays within one group of
// SMs, so this is less than the CTAs that fit divided by the cluster's size, by what the groups' sizes leave over: with four
// CTAs an SM of 148, 71 clusters of 8, not 74. (0 where not even one fits.) One object per kernel, block and `smem`.
struct ClusterFit {
    std::atomic<int> known[64][4] = {};  // [device][lg]: the count and one
    template <typename K>
    cudaError_t count(K* kernel, int device, int lg, dim3 block, size_t smem, int* n) {
        if (device < 0 || device >= 64 || lg < 0 || lg > 3) return cudaErrorInvalidValue;
        const int have = known[device][lg].load(std::memory_order_relaxed);
        if (have > 0) return *n = have - 1, cudaSuccess;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(1u << lg);
        cfg.blockDim = block;
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 1u << lg;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const cudaError_t e = cudaOccupancyMaxActiveClusters(n, kernel, &cfg);
        if (e == cudaSuccess) known[device][lg].store(*n + 1, std::memory_order_relaxed);
        return e;
    }
};

// launch_pdl (common.cuh: its rule holds here too) with clusters of `cluster` CTAs along x. Every kernel over the paged cache
// goes through one of the two and waits before it reads anything, so that the launches of a step's calls overlap. What it
// reads may have been written while it was already resident, so its pointers are not __restrict__: the compiler would turn
// their loads into non-coherent ones, which ask for memory that nobody writes during the kernel.
template <typename... KArgs, typename... Args>
inline void launch_cluster(void (*kernel)(KArgs...), int cluster, dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    cfg.numAttrs = 0;
    if (pdl_enabled()) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster;
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);  // an error surfaces in LAUNCH_CHECK's cudaGetLastError
}

// pairs of halves; a NaN on either side stays
__device__ __forceinline__ unsigned min_nan2(unsigned a, unsigned b) {
    unsigned r;
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ unsigned max_nan2(unsigned a, unsigned b) {
    unsigned r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned cluster_size() {
    unsigned r;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}
// All threads of the cluster; writes before it (global and shared) are visible behind it.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same barrier in two halves, without an order of memory: behind the wait every CTA of the cluster has started.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
// Address of a shared variable of this CTA in the CTA `rank` of the cluster.
__device__ __forceinline__ unsigned cluster_addr(const void* p, unsigned rank) {
    unsigned a = (unsigned)__cvta_generic_to_shared(p), r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ uint4 cluster_load_u32x4(unsigned addr) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_store(unsigned addr, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }
__device__ __forceinline__ void cluster_store(unsigned addr, float4 v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void cluster_store(unsigned addr, int v) { asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ void cluster_store(unsigned addr, unsigned v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ void cluster_store(unsigned addr, unsigned long long v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
#endif
