// Pages of a residency pool on the device: fork, copy, free and compact
// (kvm_pool_fork, kvm_pool_copy, kvm_pool_free, kvm_pool_compact).
//
// Each call is a plan (one small CTA per row: the new tables and, per group, a
// list of moves {source slot, destination slot}) and a copy that walks the lists
// on the device, so no count is read back. A group is one source row and the rows
// its pages go to. The copy is bound by HBM: every page is read once and written
// once per destination. 16 KiB chunks go through shared memory with bulk TMA copies
// (global -> shared, then shared -> each destination); no registers hold data in
// flight, so one CTA of kPcStages warps per SM, each with one chunk on its way, keeps
// the memory busy. One thread for all stages spent more on finding the chunks'
// addresses than the copies took (333 items of 512 KiB: 108 us against 61). 61 us are
// 0.88 of the measured copy rate; a fork of 16 rows of 34 pages of 1 MiB into three
// rows each (2.2 GB read and written) takes 380 us, 0.90.
#pragma once
#include "stagein.cuh"

namespace kvmb {

constexpr uint32_t kPcGroups = 1024;  // groups (rows, items) per launch; more are launched in turn
constexpr uint32_t kPcChunk = 16384;
constexpr uint32_t kPcStages = 12;
constexpr int kPcPlanThreads = 256;
constexpr int kPcPlainThreads = 256;
constexpr int kPcThreads = int(kPcStages) * 32;
constexpr uint32_t kPcSmem = kPcStages * kPcChunk + kPcStages * 8 + (kPcGroups + 1) * 4;

struct PageGroups {
    uint32_t n, n_dst;
    uint32_t src_row[kPcGroups];    // of group g
    uint32_t first[kPcGroups + 1];  // group g's destinations: dst_row[first[g]] .. dst_row[first[g + 1] - 1]
    uint32_t dst_row[kPcGroups];
};

struct PageItems {
    uint32_t n, n_rows;
    kvm_page_copy item[kPcGroups];  // by destination row, then in the caller's order
    uint32_t first[kPcGroups + 1];  // items of the r-th destination row
};

struct PageRows {
    uint32_t n;
    uint32_t row[kPcGroups];
};

// Tables of the destination rows, and each group's moves (by the CTA of its first
// destination): the source's slots whose page is below page_end.
__global__ void __launch_bounds__(kPcPlanThreads) fork_plan_kernel(PoolView pool, const __grid_constant__ PageGroups gr,
                                                                   uint32_t page_end, int2* moves, uint32_t* n_moves) {
    grid_release();
    __shared__ uint32_t warp_sums[32];
    const int tid = threadIdx.x;
    const uint32_t d = blockIdx.x, dst = gr.dst_row[d];
    uint32_t lo = 0, hi = gr.n;  // the group with first[g] <= d < first[g + 1]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (gr.first[mid] <= d) lo = mid;
        else hi = mid;
    }
    const uint32_t g = lo, src = gr.src_row[g];
    const int32_t* s_slot = pool.slot_of + uint64_t(src) * pool.pages;
    const int32_t* s_page = pool.page_of + uint64_t(src) * pool.slots;
    int32_t* d_slot = pool.slot_of + uint64_t(dst) * pool.pages;
    int32_t* d_page = pool.page_of + uint64_t(dst) * pool.slots;
    for (uint32_t p = tid; p < pool.pages; p += blockDim.x) d_slot[p] = p < page_end ? s_slot[p] : -1;
    uint32_t n = 0;
    for (uint32_t base = 0; base < pool.slots; base += blockDim.x) {
        const uint32_t s = base + tid;
        const int32_t p = s < pool.slots ? s_page[s] : -1;
        const bool keep = p >= 0 && uint32_t(p) < page_end;
        if (s < pool.slots) d_page[s] = keep ? p : -1;
        if (d == gr.first[g]) {
            uint32_t pre;
            const uint32_t tot = block_exclusive_scan(keep ? 1u : 0u, warp_sums, &pre);
            if (keep) moves[uint64_t(g) * pool.slots + n + pre] = make_int2(int(s), int(s));
            n += tot;
        }
    }
    if (tid == 0) {
        if (d == gr.first[g]) n_moves[g] = n;
        pool.n_restore[dst] = 0;
    }
}

// Slots of the items of one destination row; moves[i] = the i-th item's {source
// slot, destination slot}, n_moves[i] = 1, or 0 where it is left out.
__global__ void __launch_bounds__(kPcPlanThreads) copy_plan_kernel(PoolView pool, const __grid_constant__ PageItems it,
                                                                   int2* moves, uint32_t* n_moves, DeviceStatus* status) {
    grid_release();
    __shared__ uint32_t warp_sums[32];
    __shared__ uint32_t free_slot[kPcPlanThreads];
    const int tid = threadIdx.x;
    const uint32_t b = it.first[blockIdx.x], e = it.first[blockIdx.x + 1];
    const uint32_t dst = it.item[b].dst_row;
    int32_t* d_slot = pool.slot_of + uint64_t(dst) * pool.pages;
    int32_t* d_page = pool.page_of + uint64_t(dst) * pool.slots;
    uint32_t scan_at = 0;  // slots before this one are taken or handed out
    for (uint32_t base = b; base < e; base += blockDim.x) {
        const uint32_t i = base + tid;
        int src_slot = -1, slot = -1;
        uint32_t page = 0;
        if (i < e) {
            const kvm_page_copy& x = it.item[i];
            page = x.dst_page;
            src_slot = pool.slot_of[uint64_t(x.src_row) * pool.pages + x.src_page];
            if (src_slot < 0) record_error(status, KVM_ERR_STALE, 110);
            else slot = d_slot[page];
        }
        const uint32_t want = (src_slot >= 0 && slot < 0) ? 1u : 0u;
        uint32_t rank;
        const uint32_t need = block_exclusive_scan(want, warp_sums, &rank);
        // The next `need` free slots, ascending.
        uint32_t got = 0;
        while (got < need && scan_at < pool.slots) {
            const uint32_t s = scan_at + tid;
            const uint32_t f = (s < pool.slots && d_page[s] < 0) ? 1u : 0u;
            uint32_t pre;
            const uint32_t tot = block_exclusive_scan(f, warp_sums, &pre);
            if (f && got + pre < need) free_slot[got + pre] = s;
            if (got + tot >= need) {
                __syncthreads();
                scan_at = free_slot[need - 1] + 1;
                got = need;
            } else {
                got += tot;
                scan_at += blockDim.x;
            }
        }
        __syncthreads();
        if (want) {
            if (rank < got) {
                slot = int(free_slot[rank]);
                d_slot[page] = slot;
                d_page[slot] = int32_t(page);
            } else {
                record_error(status, KVM_ERR_BUDGET_EXCEEDED, 111);
            }
        }
        if (i < e) {
            const bool ok = src_slot >= 0 && slot >= 0;
            moves[i] = make_int2(src_slot, slot);
            n_moves[i] = ok ? 1u : 0u;
        }
        __syncthreads();  // the tables written above are read by the next round
    }
    if (tid == 0) pool.n_restore[dst] = 0;
}

__global__ void __launch_bounds__(kPcPlanThreads) free_kernel(PoolView pool, const __grid_constant__ PageRows rows,
                                                              uint32_t row_at, const uint32_t* ids, const uint32_t* counts,
                                                              uint32_t stride, DeviceStatus* status) {
    const uint32_t row = rows.row[blockIdx.x], at = row_at + blockIdx.x;
    int32_t* slot_of = pool.slot_of + uint64_t(row) * pool.pages;
    int32_t* page_of = pool.page_of + uint64_t(row) * pool.slots;
    uint32_t n = counts[at];
    if (n > stride) {
        if (threadIdx.x == 0) record_error(status, KVM_ERR_INVALID_ARGUMENT, 112);
        n = stride;
    }
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const uint32_t p = ids[uint64_t(at) * stride + i];
        if (p >= pool.pages) {
            record_error(status, KVM_ERR_INVALID_ARGUMENT, 113);
            continue;
        }
        const int32_t s = slot_of[p];  // a repeated page: both threads write the same, or the later one finds -1
        if (s >= 0) {
            slot_of[p] = -1;
            page_of[s] = -1;
        }
    }
    if (threadIdx.x == 0) pool.n_restore[row] = 0;
}

// With c resident pages, the k-th resident slot >= c goes to the k-th free slot < c.
__global__ void __launch_bounds__(kPcPlanThreads) compact_plan_kernel(PoolView pool, const __grid_constant__ PageGroups gr,
                                                                      int2* moves, uint32_t* n_moves, uint32_t* used) {
    grid_release();
    __shared__ uint32_t warp_sums[32];
    __shared__ uint32_t sh_n;
    const int tid = threadIdx.x;
    const uint32_t g = blockIdx.x, row = gr.src_row[g];
    int32_t* slot_of = pool.slot_of + uint64_t(row) * pool.pages;
    int32_t* page_of = pool.page_of + uint64_t(row) * pool.slots;
    int2* list = moves + uint64_t(g) * pool.slots;
    if (tid == 0) sh_n = 0;
    __syncthreads();
    uint32_t mine = 0;
    for (uint32_t s = tid; s < pool.slots; s += blockDim.x) mine += page_of[s] >= 0;
    if (mine) atomicAdd(&sh_n, mine);
    __syncthreads();
    const uint32_t c = sh_n;
    uint32_t holes = 0, movers = 0;
    for (uint32_t base = 0; base < pool.slots; base += blockDim.x) {
        const uint32_t s = base + tid;
        const bool held = s < pool.slots && page_of[s] >= 0;
        const uint32_t hole = (s < c && !held) ? 1u : 0u, mover = (s >= c && held) ? 1u : 0u;
        uint32_t pre;
        uint32_t tot = block_exclusive_scan(hole, warp_sums, &pre);
        if (hole) list[holes + pre].y = int(s);
        holes += tot;
        tot = block_exclusive_scan(mover, warp_sums, &pre);
        if (mover) list[movers + pre].x = int(s);
        movers += tot;
    }
    __syncthreads();
    for (uint32_t k = tid; k < movers; k += blockDim.x) {  // holes == movers
        const int2 m = list[k];
        const int32_t p = page_of[m.x];
        page_of[m.x] = -1;
        page_of[m.y] = p;
        slot_of[p] = m.y;
    }
    if (tid == 0) {
        n_moves[g] = movers;
        if (used) used[g] = c;
        pool.n_restore[row] = 0;
    }
}

// The pages of the groups' move lists, chunk by chunk. Group g's list starts at
// moves + g * list_stride.
struct PageCopy {
    GatherLayout lay;
    const int2* moves;
    const uint32_t* n_moves;
    uint32_t list_stride;
    uint32_t chunk;      // bytes per chunk
    uint32_t chunks[2];  // chunks of a page of each plane
    DeviceStatus* status;
};

// Exclusive prefix of the groups' move counts into sums[0 .. n] (one warp).
__device__ __forceinline__ void page_prefix(const PageGroups& gr, const uint32_t* n_moves, uint32_t* sums) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t total = 0;
    for (uint32_t base = 0; base < gr.n; base += 32) {
        const uint32_t g = base + lane;
        uint32_t v = g < gr.n ? n_moves[g] : 0, x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= uint32_t(o)) x += y;
        }
        if (g < gr.n) sums[g] = total + x - v;
        total += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) sums[gr.n] = total;
}

struct PageChunk {
    uint32_t g;
    int2 move;
    uint32_t plane, offset, bytes;
};

__device__ __forceinline__ PageChunk page_chunk(const PageGroups& gr, const PageCopy& pc, const uint32_t* sums,
                                                uint64_t item) {
    const uint32_t per = pc.chunks[0] + pc.chunks[1];
    const uint32_t page = uint32_t(item / per);
    uint32_t c = uint32_t(item - uint64_t(page) * per);
    uint32_t lo = 0, hi = gr.n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (sums[mid] <= page) lo = mid;
        else hi = mid;
    }
    PageChunk x;
    x.g = lo;
    x.move = pc.moves[uint64_t(lo) * pc.list_stride + (page - sums[lo])];
    x.plane = c >= pc.chunks[0];
    if (x.plane) c -= pc.chunks[0];
    x.offset = c * pc.chunk;
    x.bytes = uint32_t(min(uint64_t(pc.chunk), pc.lay.bytes[x.plane] - x.offset));
    return x;
}

__device__ __forceinline__ uint8_t* page_at(const GatherLayout& lay, uint32_t plane, uint32_t row, uint32_t slot) {
    return lay.dev_base[plane] + uint64_t(row) * lay.dev_row_stride[plane] + uint64_t(slot) * lay.dev_slot_stride[plane];
}

// One thread of each warp owns a stage: load, store to every destination, next chunk.
// The address of a chunk (a search in shared memory and a load of its move) is worked
// out while the chunk before it is on its way.
__global__ void __launch_bounds__(kPcThreads) page_copy_kernel(const __grid_constant__ PageGroups gr,
                                                               const __grid_constant__ PageCopy pc) {
    extern __shared__ __align__(128) uint8_t ring[];
    uint64_t* full = reinterpret_cast<uint64_t*>(ring + kPcStages * kPcChunk);
    uint32_t* sums = reinterpret_cast<uint32_t*>(full + kPcStages);
    const uint32_t warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < kPcStages; ++s) mbar_init(&full[s], 1);
        mbar_fence_init();
    }
    grid_wait();
    if (warp == 0) page_prefix(gr, pc.n_moves, sums);
    __syncthreads();
    if (threadIdx.x & 31) return;
    // The plan's tables and lists are generic-proxy writes of another kernel; the pages are
    // read and written by the async proxy only.
    asm volatile("fence.proxy.async;" ::: "memory");
    const uint64_t items = uint64_t(sums[gr.n]) * (pc.chunks[0] + pc.chunks[1]);
    const uint64_t step = uint64_t(gridDim.x) * kPcStages;
    const uint64_t policy = policy_evict_first();
    uint8_t* stage = ring + warp * kPcChunk;
    uint64_t i = blockIdx.x + uint64_t(warp) * gridDim.x;
    if (i >= items) return;
    PageChunk x = page_chunk(gr, pc, sums, i);
    for (uint32_t phase = 0;; phase ^= 1) {
        mbar_arrive_expect_tx(&full[warp], x.bytes);
        bulk_g2s(stage, page_at(pc.lay, x.plane, gr.src_row[x.g], uint32_t(x.move.x)) + x.offset, x.bytes, &full[warp], policy);
        const PageChunk y = x;
        i += step;
        if (i < items) x = page_chunk(gr, pc, sums, i);
        if (!mbar_wait(&full[warp], phase)) {
            record_error(pc.status, KVM_ERR_TIMEOUT, 114);
            mbar_wait(&full[warp], phase);  // the load lands before the shared memory is freed
            break;
        }
        for (uint32_t d = gr.first[y.g]; d < gr.first[y.g + 1]; ++d)
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(
                             page_at(pc.lay, y.plane, gr.dst_row[d], uint32_t(y.move.y)) + y.offset),
                         "r"(smem_u32(stage)), "r"(y.bytes)
                         : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        if (i >= items) break;
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// Pages whose addresses or size are no multiples of 16 bytes.
__global__ void __launch_bounds__(kPcPlainThreads) page_copy_plain_kernel(const __grid_constant__ PageGroups gr,
                                                                          const __grid_constant__ PageCopy pc) {
    __shared__ uint32_t sums[kPcGroups + 1];
    grid_wait();
    if (threadIdx.x < 32) page_prefix(gr, pc.n_moves, sums);
    __syncthreads();
    const uint64_t items = uint64_t(sums[gr.n]) * (pc.chunks[0] + pc.chunks[1]);
    for (uint64_t i = blockIdx.x; i < items; i += gridDim.x) {
        const PageChunk x = page_chunk(gr, pc, sums, i);
        const uint8_t* src = page_at(pc.lay, x.plane, gr.src_row[x.g], uint32_t(x.move.x)) + x.offset;
        for (uint32_t d = gr.first[x.g]; d < gr.first[x.g + 1]; ++d)
            copy_item(src, page_at(pc.lay, x.plane, gr.dst_row[d], uint32_t(x.move.y)) + x.offset, x.bytes);
    }
}

}  // namespace kvmb
