// Attention of a few rows over a cache: a sliding window with sinks over a dense
// cache (kvm_window_attention) and a tree of drafted tokens over the pages of a
// residency pool (kvm_tree_attention).
//
//   out_i = sum_t exp(s_it - lse_i) V_t,   s_it = scale <q_i, K_t>,
//   lse_i = log sum_t exp(s_it)            over the keys t that row i sees
//
// attend_mma_kernel: one CTA of four warps per (sequence, KV head, M tile, key
// chunk). The G query heads of a KV head are packed with the rows (packed row
// m = row * G + head), so a key is read once per KV head and not once per query
// head. Keys come in tiles of 64 through a ring of cp.async stages; the four
// warps split an M tile of 16 * WM packed rows and the tile's keys between them
// (WM = 1: each warp takes 16 of the 64 keys, its own running max, sum and output
// rows, merged at the end; WM = 4: each warp takes 16 rows and every key). One
// pass: running max and sum in the log2 domain in 32 bits, P rounded to the
// operand type for the second product (its error, half a step of that type
// relative, is that of the output's own rounding).
//
// Few rows are bound by the reading of K and V: the key range is cut into
// `splits` chunks so that every SM reads, and attend_combine_kernel joins the
// chunks' (max, sum, unnormalised rows).
//
// Measured (device time, joining pass included): one row, 8 lanes, 4,224 keys, 40 / 8 heads,
// head_dim 128: 29.5 us, 4.7 TB/s, 0.73 of the measured copy rate; one lane of 1,027 keys, 24 / 4
// heads, head_dim 256: 9.1 us, two launches and a chain of dependent loads. A tile of 64 keys of
// head_dim 256 takes 2.6 us (four warps, one per scheduler, bound by instruction latency): long
// page lists go to the tcgen05 kernel even for one row.
#pragma once
#include "common.cuh"

namespace kvmb {

constexpr int kAtThreads = 128;
constexpr int kAtKeys = 64;    // keys per tile
constexpr int kAtTable = 512;  // page entries held in shared memory at a time
constexpr int kAtWindow = 0, kAtTree = 1;
constexpr float kAtLn2 = 0.6931471805599453f;

struct AttendParams {
    const uint8_t* q;
    uint64_t q_seq, q_row, q_head;  // byte strides
    uint8_t* out;
    uint64_t o_seq, o_row, o_head;
    float* lse;  // [seqs][width][q_heads] or null
    uint32_t seqs, width, q_heads, kv_heads, group;
    uint32_t m_tiles, splits;
    uint64_t g_magic;  // m / group = (m * g_magic) >> g_shift for m < 2^31
    uint32_t g_shift;
    float scale_log2;
    // Dense keys: the window's cache, or the tree's tail.
    const uint8_t *k, *v;
    uint64_t k_seq, k_tok, k_head, v_seq, v_tok, v_head;
    uint32_t capacity;          // tokens per sequence
    const uint32_t* seq_rows;   // rows used per sequence, or null (width)
    // Window.
    uint64_t base;
    const uint64_t* seq_base;   // or null (base)
    uint32_t window, sinks;
    // Tree: pages of the pool.
    const uint8_t *pk, *pv;
    uint64_t pk_row, pk_slot, pk_tok, pk_head, pv_row, pv_slot, pv_tok, pv_head;
    int32_t pk_type, pv_type;
    uint32_t pk_bytes, pv_bytes;  // bytes of one row of one head
    uint32_t pk_gran, pv_gran;    // copy granularity of quantised rows (4, 8 or 16)
    const int32_t *slot_of, *page_of;
    uint32_t pool_pages, pool_slots, row0, row_step;
    const uint32_t *sel_ids, *sel_n;
    uint32_t sel_stride, sel_width, page_tokens;
    uint64_t pt_magic;  // u / page_tokens = (u * pt_magic) >> pt_shift for u < 2^31
    uint32_t pt_shift;
    uint64_t tokens;
    const uint64_t* seq_tokens;  // or null (tokens)
    uint32_t recent;
    const uint32_t* seq_recent;  // or null (recent)
    const uint32_t* tree;        // or null (chain)
    uint64_t tree_seq;           // words between sequences' trees
    uint32_t tree_words;         // words per node
    float* part_o;               // [splits][seqs][width][q_heads][D]
    float2* part_ml;             // [splits][seqs][width][q_heads] {max (log2 units), sum}
    DeviceStatus* status;
};

__device__ __forceinline__ void at_cp16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void at_cp8(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(valid ? 8 : 0) : "memory");
}
__device__ __forceinline__ void at_cp4(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void at_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void at_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void at_ldsm4(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void at_ldsm4t(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <bool BF16>
__device__ __forceinline__ void at_mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool BF16>
__device__ __forceinline__ uint32_t at_pack(float a, float b) {
    if constexpr (BF16) {
        __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&h);
    } else {
        __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&h);
    }
}
template <bool BF16>
__device__ __forceinline__ float2 at_unpack(uint32_t w) {
    if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<__half2*>(&w));
}

// Whether one of two packed 16-bit values is infinite or NaN (exponent all ones).
template <bool BF16>
__device__ __forceinline__ bool at_nonfinite(uint32_t w) {
    constexpr uint32_t e = BF16 ? 0x7F80u : 0x7C00u;
    return (w & e) == e || ((w >> 16) & e) == e;
}

// Byte offset of 16-byte chunk c of row r in a tile of D-element rows: chunks are
// permuted by the row so that 8 rows of one chunk (ldmatrix) meet 8 bank groups.
template <int D>
__device__ __forceinline__ uint32_t at_off(uint32_t r, uint32_t c) {
    return r * (D * 2) + ((c ^ (r & 7)) << 4);
}

// Two codes (bytes at bits 0-7 and 16-23 of x, the rest zero) as packed 16-bit
// numbers, exactly: 8-bit two's complement, or 4-bit with offset 8.
template <bool BF16>
__device__ __forceinline__ uint32_t at_codes8(uint32_t x) {
    if constexpr (BF16) {
        // 128 + low 7 bits, minus 128 or (sign) 256: all exact in 8 bits of mantissa.
        const uint32_t lo = (x & 0x007F007Fu) | 0x43004300u, hi = (x & 0x00800080u) | 0x43004300u;
        const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&lo), *reinterpret_cast<const __nv_bfloat162*>(&hi));
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const uint32_t u = (x ^ 0x00800080u) | 0x64006400u, b = 0x64806480u;  // 1024 + (code + 128), 1152
        const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&u), *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}
template <bool BF16>
__device__ __forceinline__ uint32_t at_codes4(uint32_t x) {
    if constexpr (BF16) {
        const uint32_t u = x | 0x43004300u, b = 0x43084308u;  // 128 + code, 136
        const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const uint32_t u = x | 0x64006400u, b = 0x64086408u;  // 1024 + code, 1032
        const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&u), *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}

// Ring stages of a variant: as many as fit beside the query tile.
__host__ __device__ constexpr uint32_t at_stage_bytes(int D, bool quant) {
    return quant ? 2u * 64u * uint32_t(D / 32 * 34) : 2u * 64u * uint32_t(D) * 2u;
}
__host__ __device__ constexpr uint32_t at_stages(int D, int WM, bool quant) {
    return (D == 256 && WM == 4 && !quant) ? 2u : 3u;
}
__host__ __device__ constexpr uint32_t at_smem_bytes(int D, int WM, bool quant) {
    // query tile, ring, (quantised: the decoded tile and its block scales), page table, merge table
    return uint32_t(16 * WM * D * 2) + at_stages(D, WM, quant) * at_stage_bytes(D, quant) +
           (quant ? 2u * 64u * uint32_t(D) * 2u + 2u * 64u * uint32_t(D / 32) * 4u : 0u) + uint32_t(kAtTable) * 8u +
           4u * 16u * uint32_t(WM) * 8u / uint32_t(WM) + 16u;
}

// A quantised V block's scale is applied to P before it is rounded (P * d, one
// rounding); in fp16 P * d is kept 2^6 higher, so that small probabilities of small
// blocks stay clear of the subnormal range. Scales above 1023 would overflow there:
// they are reported as KVM_ERR_NONFINITE.
constexpr float kAtLift = 64.f;

template <int D, int WM, bool BF16, int MODE, bool QUANT>
__global__ void __launch_bounds__(kAtThreads) attend_mma_kernel(const __grid_constant__ AttendParams P) {
    constexpr int WK = 4 / WM;       // warps that share an M slice, each with its own keys
    constexpr int KW = kAtKeys / WK; // keys per warp
    constexpr int NT = KW / 8;       // 8-key accumulator tiles of S
    constexpr int CH = D / 8;        // 16-byte chunks of a row
    constexpr int M = 16 * WM;
    constexpr uint32_t ST = at_stages(D, WM, QUANT);
    constexpr uint32_t kStage = at_stage_bytes(D, QUANT);
    constexpr uint32_t kHalf = kStage / 2;  // V behind K
    constexpr uint32_t kTile = 64u * D * 2u;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* qs = smem;
    uint8_t* ring = qs + M * D * 2;
    uint8_t* dec = ring + ST * kStage;  // decoded K tile, V tile (QUANT)
    float* scales = reinterpret_cast<float*>(dec + (QUANT ? 2 * kTile : 0));  // [2][64][D / 32]
    int2* table = reinterpret_cast<int2*>(reinterpret_cast<uint8_t*>(scales) + (QUANT ? 2 * 64 * (D / 32) * 4 : 0));
    float2* sm_ml = reinterpret_cast<float2*>(table + kAtTable);  // [WK][M]

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int wm = warp % WM, wk = warp / WM;
    // Unit: M tiles fastest (they read the same keys at about the same time), then key chunks.
    uint32_t u = blockIdx.x;
    const uint32_t mt = u % P.m_tiles;
    u /= P.m_tiles;
    const uint32_t split = u % P.splits;
    u /= P.splits;
    const uint32_t h = u % P.kv_heads, b = u / P.kv_heads;
    const uint32_t G = P.group;
    const uint32_t rows = P.seq_rows ? __ldg(P.seq_rows + b) : P.width;
    if (rows > P.width) {
        if (tid == 0) record_error(P.status, KVM_ERR_LENGTH, 106);
        return;
    }
    const uint32_t m0 = mt * M, m_end = rows * G;  // packed rows [m0, min(m0 + M, m_end))
    if (m0 >= m_end) return;
    const uint32_t i0 = m0 / G, i1 = min(m0 + M - 1, m_end - 1) / G;  // rows of this M tile

    // ---- the keys of this unit: `nt` tiles ----
    uint32_t nt, n_first;        // tiles in all; sink tiles / page tiles, which come first
    uint32_t p0 = 0, p1 = 0, lo = 0, hi = 0, few = 0;     // window
    uint32_t n_list = 0, n_keys = 0, recent = 0, tail = 0;  // tree
    uint64_t tokens = 0;
    const uint8_t *kd, *vd;      // dense keys of this sequence and head
    const int32_t *slot_of = nullptr, *page_of = nullptr;
    const uint32_t* ids = nullptr;
    const uint8_t *pk = nullptr, *pv = nullptr;
    kd = P.k + uint64_t(b) * P.k_seq + uint64_t(h) * P.k_head;
    vd = P.v + uint64_t(b) * P.v_seq + uint64_t(h) * P.v_head;
    if constexpr (MODE == kAtWindow) {
        const uint64_t base = P.seq_base ? __ldg(reinterpret_cast<const unsigned long long*>(P.seq_base + b)) : P.base;
        if (base > P.capacity || rows > P.capacity - base) {  // keys past the cache: the sequence is left out
            if (tid == 0) record_error(P.status, KVM_ERR_LENGTH, 100);
            return;
        }
        p0 = uint32_t(base) + i0;
        p1 = uint32_t(base) + i1;
        hi = p1 + 1;
        lo = P.window == 0 ? hi : (p0 + 1 > P.window ? p0 + 1 - P.window : 0);
        few = min(P.sinks, lo);
        n_first = (few + kAtKeys - 1) / kAtKeys;
        nt = n_first + (hi - lo + kAtKeys - 1) / kAtKeys;
    } else {
        const uint32_t row = P.row0 + b * P.row_step;
        slot_of = P.slot_of + uint64_t(row) * P.pool_pages;
        page_of = P.page_of + uint64_t(row) * P.pool_slots;
        tokens = P.seq_tokens ? __ldg(reinterpret_cast<const unsigned long long*>(P.seq_tokens + b)) : P.tokens;
        recent = P.seq_recent ? __ldg(P.seq_recent + b) : P.recent;
        if (recent > P.capacity || rows > P.capacity - recent) {
            if (tid == 0) record_error(P.status, KVM_ERR_LENGTH, 101);
            return;
        }
        tail = recent + rows;
        if (P.sel_ids) {
            ids = P.sel_ids + uint64_t(b) * P.sel_stride;
            n_list = __ldg(P.sel_n + b);
            if (n_list > P.sel_width) {
                if (tid == 0) record_error(P.status, KVM_ERR_INVALID_ARGUMENT, 102);
                n_list = P.sel_width;
            }
        } else {
            n_list = P.pool_slots;
        }
        n_keys = n_list * P.page_tokens;
        n_first = (n_keys + kAtKeys - 1) / kAtKeys;
        nt = n_first + (tail + kAtKeys - 1) / kAtKeys;
        pk = P.pk + uint64_t(row) * P.pk_row + uint64_t(h) * P.pk_head;
        pv = P.pv + uint64_t(row) * P.pv_row + uint64_t(h) * P.pv_head;
    }
    const uint32_t tb = uint32_t(uint64_t(nt) * split / P.splits), te = uint32_t(uint64_t(nt) * (split + 1) / P.splits);

    // ---- the query tile ----
    for (int e = tid; e < M * CH; e += kAtThreads) {
        const uint32_t r = e / CH, c = e % CH, m = m0 + r;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (m < m_end) {
            const uint32_t i = m / G, g = m - i * G;
            x = __ldg(reinterpret_cast<const uint4*>(P.q + uint64_t(b) * P.q_seq + uint64_t(i) * P.q_row +
                                                     uint64_t(h * G + g) * P.q_head) + c);
        }
        *reinterpret_cast<uint4*>(qs + at_off<D>(r, c)) = x;
    }

    auto page_div = [&](uint32_t x) { return uint32_t((uint64_t(x) * P.pt_magic) >> P.pt_shift); };
    // Entries [e0, e0 + kAtTable) of the page list: {slot, tokens held}; {., 0} where the page is absent.
    uint32_t e0 = 0xffffffffu;
    auto fill_table = [&](uint32_t first) {
        e0 = first;
        for (uint32_t i = tid; i < uint32_t(kAtTable); i += kAtThreads) {
            const uint32_t e = first + i;
            int2 ent = make_int2(0, 0);
            if (e < n_list) {
                int page, slot;
                if (ids) {
                    const uint32_t id = __ldg(ids + e);
                    page = id < P.pool_pages ? int(id) : -1;
                    slot = page >= 0 ? slot_of[page] : -1;
                    if (page < 0) record_error(P.status, KVM_ERR_INVALID_ARGUMENT, 103);
                    else if (slot < 0 || slot >= int(P.pool_slots)) {
                        record_error(P.status, KVM_ERR_STALE, 104);
                        page = -1;
                    }
                } else {
                    slot = int(e);
                    page = page_of[e];
                }
                if (page >= 0) {
                    const uint64_t start = uint64_t(page) * P.page_tokens;
                    const uint64_t held = tokens > start ? tokens - start : 0;
                    ent = make_int2(slot, int(min(held, uint64_t(P.page_tokens))));
                }
            }
            table[i] = ent;
        }
    };
    // Last list entry that tile t touches.
    auto last_entry = [&](uint32_t t) { return page_div(min(t * kAtKeys + kAtKeys - 1, n_keys - 1)); };

    // Starts the copies of tile t into ring stage s.
    auto issue = [&](uint32_t t, uint32_t s) {
        const uint32_t kdst = smem_u32(ring + s * kStage), vdst = kdst + kHalf;
        if (!QUANT || MODE == kAtWindow) {
#pragma unroll 4
            for (int it = 0; it < CH / 2; ++it) {
                const uint32_t e = tid + it * kAtThreads, r = e / CH, c = e % CH;
                const uint8_t *ks, *vs;
                bool valid;
                if constexpr (MODE == kAtWindow) {
                    const uint32_t tok = t < n_first ? t * kAtKeys + r : lo + (t - n_first) * kAtKeys + r;
                    valid = tok < (t < n_first ? few : hi);
                    const uint32_t tk = valid ? tok : 0;
                    ks = kd + uint64_t(tk) * P.k_tok;
                    vs = vd + uint64_t(tk) * P.v_tok;
                } else if (t < n_first) {
                    const uint32_t x = t * kAtKeys + r, en = page_div(x), o = x - en * P.page_tokens;
                    const int2 ent = x < n_keys ? table[en - e0] : make_int2(0, 0);
                    valid = int(o) < ent.y;
                    ks = pk + uint64_t(uint32_t(ent.x)) * P.pk_slot + uint64_t(valid ? o : 0) * P.pk_tok;
                    vs = pv + uint64_t(uint32_t(ent.x)) * P.pv_slot + uint64_t(valid ? o : 0) * P.pv_tok;
                } else {
                    const uint32_t x = (t - n_first) * kAtKeys + r;
                    valid = x < tail;
                    ks = kd + uint64_t(valid ? x : 0) * P.k_tok;
                    vs = vd + uint64_t(valid ? x : 0) * P.v_tok;
                }
                at_cp16(kdst + at_off<D>(r, c), ks + c * 16, valid);
                at_cp16(vdst + at_off<D>(r, c), vs + c * 16, valid);
            }
        } else {
            // Quantised rows as stored, back to back.
            auto plane = [&](uint32_t dst, const uint8_t* src, uint64_t slot_stride, uint64_t tok_stride, uint32_t rb,
                             uint32_t gran) {
                const uint32_t per = rb / gran;
                for (uint32_t e = tid; e < kAtKeys * per; e += kAtThreads) {
                    const uint32_t r = e / per, c = (e - r * per) * gran;
                    const uint32_t x = t * kAtKeys + r, en = page_div(x), o = x - en * P.page_tokens;
                    const int2 ent = x < n_keys ? table[en - e0] : make_int2(0, 0);
                    const bool valid = int(o) < ent.y;
                    const uint8_t* p = src + uint64_t(uint32_t(ent.x)) * slot_stride + uint64_t(valid ? o : 0) * tok_stride + c;
                    if (gran == 16) at_cp16(dst + r * rb + c, p, valid);
                    else if (gran == 8) at_cp8(dst + r * rb + c, p, valid);
                    else at_cp4(dst + r * rb + c, p, valid);
                }
            };
            plane(kdst, pk, P.pk_slot, P.pk_tok, P.pk_bytes, P.pk_gran);
            plane(vdst, pv, P.pv_slot, P.pv_tok, P.pv_bytes, P.pv_gran);
        }
    };

    // What tile t holds: 0 nothing, 1 every key visible to every row, 2 keys to be masked.
    auto state_of = [&](uint32_t t) -> int {
        if constexpr (MODE == kAtWindow) {
            const uint32_t a = t < n_first ? t * kAtKeys : lo + (t - n_first) * kAtKeys;
            const uint32_t end = t < n_first ? few : hi;
            return a + kAtKeys <= end && a + kAtKeys - 1 <= p0 && (a + kAtKeys <= P.sinks || p1 - a < P.window) ? 1 : 2;
        } else {
            if (t >= n_first) return (t - n_first + 1) * kAtKeys <= recent ? 1 : 2;
            const uint32_t a = page_div(t * kAtKeys), z = last_entry(t);
            bool all = t * kAtKeys + kAtKeys <= n_keys, none = true;
            for (uint32_t e = a; e <= z; ++e) {
                const int cnt = table[e - e0].y;
                all = all && cnt == int(P.page_tokens);
                none = none && cnt == 0;
            }
            return none ? 0 : all ? 1 : 2;
        }
    };
    // Whether row i (position p0 + i - i0) sees key j of tile t.
    auto sees = [&](uint32_t i, uint32_t t, uint32_t j) -> bool {
        if constexpr (MODE == kAtWindow) {
            const uint32_t tok = t < n_first ? t * kAtKeys + j : lo + (t - n_first) * kAtKeys + j;
            const uint32_t p = p0 + (i - i0);
            return tok < (t < n_first ? few : hi) && tok <= p && (p - tok < P.window || tok < P.sinks);
        } else {
            if (t < n_first) {
                const uint32_t x = t * kAtKeys + j;
                if (x >= n_keys) return false;
                const uint32_t en = page_div(x);
                return int(x - en * P.page_tokens) < table[en - e0].y;
            }
            const uint32_t x = (t - n_first) * kAtKeys + j;
            if (x < recent) return true;
            const uint32_t n = x - recent;
            if (n >= rows) return false;
            if (!P.tree) return n <= i;
            return (__ldg(P.tree + uint64_t(b) * P.tree_seq + uint64_t(i) * P.tree_words + (n >> 5)) >> (n & 31)) & 1;
        }
    };

    // ---- running state of this warp's 16 rows over its keys ----
    const int qr = lane >> 2, qc = lane & 3;  // accumulator row (and + 8) and column pair
    uint32_t ri[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) ri[x] = min((m0 + wm * 16 + qr + 8 * x) / G, rows - 1);
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
    float mx[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const float c2 = P.scale_log2;
    const uint32_t qbase = smem_u32(qs) + 0;

    // One tile whose K and V rows (16-bit numbers, or exact codes with block scales) are at ks and vs.
    auto compute = [&](uint32_t t, int st, uint8_t* ktile, uint8_t* vtile, bool codes) {
        const uint32_t ks = smem_u32(ktile), vs = smem_u32(vtile);
        float s[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[j][k] = 0.f;
        const uint32_t krow = wk * KW;
        // S = Q K^T
        if (!QUANT || !codes) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                uint32_t a[4];
                at_ldsm4(qbase + at_off<D>(wm * 16 + (lane & 15), kk * 2 + (lane >> 4)), a);
#pragma unroll
                for (int j = 0; j < NT; j += 2) {
                    uint32_t bb[4];  // keys 8j .. 8j + 15, dims 16kk .. + 15
                    at_ldsm4(ks + at_off<D>(krow + j * 8 + (lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)), bb);
                    at_mma<BF16>(s[j], a, bb[0], bb[1]);
                    at_mma<BF16>(s[j + 1], a, bb[2], bb[3]);
                }
            }
        } else {
            const float* kscale = scales;
#pragma unroll
            for (int blk = 0; blk < D / 32; ++blk) {
                float acc[NT][4];
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[j][k] = 0.f;
#pragma unroll
                for (int kk = 2 * blk; kk < 2 * blk + 2; ++kk) {
                    uint32_t a[4];
                    at_ldsm4(qbase + at_off<D>(wm * 16 + (lane & 15), kk * 2 + (lane >> 4)), a);
#pragma unroll
                    for (int j = 0; j < NT; j += 2) {
                        uint32_t bb[4];
                        at_ldsm4(ks + at_off<D>(krow + j * 8 + (lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)), bb);
                        at_mma<BF16>(acc[j], a, bb[0], bb[1]);
                        at_mma<BF16>(acc[j + 1], a, bb[2], bb[3]);
                    }
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const float d0 = kscale[(krow + j * 8 + qc * 2) * (D / 32) + blk];
                    const float d1 = kscale[(krow + j * 8 + qc * 2 + 1) * (D / 32) + blk];
                    s[j][0] += acc[j][0] * d0;
                    s[j][1] += acc[j][1] * d1;
                    s[j][2] += acc[j][2] * d0;
                    s[j][3] += acc[j][3] * d1;
                }
            }
        }
        if (st == 2) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (!sees(ri[k >> 1], t, krow + j * 8 + qc * 2 + (k & 1))) s[j][k] = -INFINITY;
        }
        // Running max; rows that have seen nothing yet subtract 0 from -inf.
        float sub[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            float v = s[0][2 * x];
#pragma unroll
            for (int j = 0; j < NT; ++j) v = fmaxf(v, fmaxf(s[j][2 * x], s[j][2 * x + 1]));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
            const float nm = fmaxf(mx[x], v * c2);
            sub[x] = nm == -INFINITY ? 0.f : nm;
            const float alpha = fast_exp2(mx[x] - sub[x]);
            mx[x] = nm;
            l[x] *= alpha;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                o[i][2 * x] *= alpha;
                o[i][2 * x + 1] *= alpha;
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                s[j][k] = fast_exp2(fmaf(s[j][k], c2, -sub[k >> 1]));
                l[k >> 1] += s[j][k];
            }
        // O += P V
        if (!QUANT || !codes) {
            bool bad = false;
            if (st == 2) {
                // Infinite or NaN values behind a mask must not reach the rows that do not see them
                // (0 * inf): such a tile is summed key by key below.
                for (int e = lane; e < KW * CH; e += 32) {
                    const uint4 x = *reinterpret_cast<const uint4*>(vtile + at_off<D>(krow + e / CH, e % CH));
                    bad = bad || at_nonfinite<BF16>(x.x) || at_nonfinite<BF16>(x.y) || at_nonfinite<BF16>(x.z) ||
                          at_nonfinite<BF16>(x.w);
                }
                bad = __any_sync(0xffffffffu, bad);
            }
            if (!bad) {
#pragma unroll
                for (int ks16 = 0; ks16 < KW / 16; ++ks16) {
                    uint32_t a[4];
                    a[0] = at_pack<BF16>(s[2 * ks16][0], s[2 * ks16][1]);
                    a[1] = at_pack<BF16>(s[2 * ks16][2], s[2 * ks16][3]);
                    a[2] = at_pack<BF16>(s[2 * ks16 + 1][0], s[2 * ks16 + 1][1]);
                    a[3] = at_pack<BF16>(s[2 * ks16 + 1][2], s[2 * ks16 + 1][3]);
#pragma unroll
                    for (int i = 0; i < D / 8; i += 2) {
                        uint32_t bb[4];
                        at_ldsm4t(vs + at_off<D>(krow + ks16 * 16 + (lane & 15), i + (lane >> 4)), bb);
                        at_mma<BF16>(o[i], a, bb[0], bb[1]);
                        at_mma<BF16>(o[i + 1], a, bb[2], bb[3]);
                    }
                }
            } else {
                for (uint32_t key = 0; key < uint32_t(KW); ++key) {
                    float pr[2] = {0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        if (uint32_t(j) == key >> 3) {
                            pr[0] = (key & 1) ? s[j][1] : s[j][0];
                            pr[1] = (key & 1) ? s[j][3] : s[j][2];
                        }
                    const int from = (lane & ~3) | int((key & 7) >> 1);
                    pr[0] = __shfl_sync(0xffffffffu, pr[0], from);
                    pr[1] = __shfl_sync(0xffffffffu, pr[1], from);
                    const bool s0 = sees(ri[0], t, krow + key), s1 = sees(ri[1], t, krow + key);
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        const float2 v2 = at_unpack<BF16>(
                            *reinterpret_cast<const uint32_t*>(vtile + at_off<D>(krow + key, i) + qc * 4));
                        if (s0) {
                            o[i][0] += pr[0] * v2.x;
                            o[i][1] += pr[0] * v2.y;
                        }
                        if (s1) {
                            o[i][2] += pr[1] * v2.x;
                            o[i][3] += pr[1] * v2.y;
                        }
                    }
                }
            }
        } else {
            const float* vscale = scales + 64 * (D / 32);
#pragma unroll
            for (int ks16 = 0; ks16 < KW / 16; ++ks16) {
                const float* sc = vscale + (krow + ks16 * 16 + qc * 2) * (D / 32);
#pragma unroll
                for (int blk = 0; blk < D / 32; ++blk) {
                    const float d0 = sc[blk], d1 = sc[D / 32 + blk], d8 = sc[8 * (D / 32) + blk], d9 = sc[9 * (D / 32) + blk];
                    uint32_t a[4];
                    a[0] = at_pack<BF16>(s[2 * ks16][0] * d0, s[2 * ks16][1] * d1);
                    a[1] = at_pack<BF16>(s[2 * ks16][2] * d0, s[2 * ks16][3] * d1);
                    a[2] = at_pack<BF16>(s[2 * ks16 + 1][0] * d8, s[2 * ks16 + 1][1] * d9);
                    a[3] = at_pack<BF16>(s[2 * ks16 + 1][2] * d8, s[2 * ks16 + 1][3] * d9);
#pragma unroll
                    for (int i = 4 * blk; i < 4 * blk + 4; i += 2) {
                        uint32_t bb[4];
                        at_ldsm4t(vs + at_off<D>(krow + ks16 * 16 + (lane & 15), i + (lane >> 4)), bb);
                        at_mma<BF16>(o[i], a, bb[0], bb[1]);
                        at_mma<BF16>(o[i + 1], a, bb[2], bb[3]);
                    }
                }
            }
        }
    };

    // ---- the pass over the tiles ----
    const uint32_t te_ring = QUANT && MODE == kAtTree ? min(te, max(n_first, tb)) : te;  // tiles that go through the ring
    if (MODE == kAtTree && tb < min(te, n_first)) fill_table(page_div(tb * kAtKeys));
    __syncthreads();
    for (uint32_t s = 0; s < ST - 1; ++s) {
        if (tb + s < te_ring) issue(tb + s, s);
        at_commit();
    }
    for (uint32_t t = tb; t < te_ring; ++t) {
        at_wait<ST - 2>();
        __syncthreads();
        const uint32_t nx = t + ST - 1;
        if (nx < te_ring) {
            if (MODE == kAtTree && nx < n_first && last_entry(nx) >= e0 + kAtTable) {
                fill_table(page_div(t * kAtKeys));
                __syncthreads();
            }
            issue(nx, (nx - tb) % ST);
        }
        at_commit();
        const int st = state_of(t);
        uint8_t* stage = ring + ((t - tb) % ST) * kStage;
        if constexpr (!QUANT) {
            if (st) compute(t, st, stage, stage + kHalf, false);
        } else {
            // Codes and block scales of this tile, then the tile.
#pragma unroll
            for (int pl = 0; pl < 2; ++pl) {
                const uint8_t* raw = stage + pl * kHalf;
                const uint32_t rb = pl ? P.pv_bytes : P.pk_bytes;
                const bool q8 = (pl ? P.pv_type : P.pk_type) == KVM_Q8_0;
                uint8_t* dst = dec + pl * kTile;
                for (int e = tid; e < kAtKeys * CH; e += kAtThreads) {
                    const uint32_t r = e / CH, c = e % CH, blk = c >> 2, part = c & 3;
                    const uint8_t* src = raw + r * rb + blk * (q8 ? 34 : 18);
                    uint4 x;
                    if (q8) {
                        const uint16_t* w = reinterpret_cast<const uint16_t*>(src + 2 + part * 8);
                        x.x = at_codes8<BF16>((w[0] & 0xffu) | (uint32_t(w[0] >> 8) << 16));
                        x.y = at_codes8<BF16>((w[1] & 0xffu) | (uint32_t(w[1] >> 8) << 16));
                        x.z = at_codes8<BF16>((w[2] & 0xffu) | (uint32_t(w[2] >> 8) << 16));
                        x.w = at_codes8<BF16>((w[3] & 0xffu) | (uint32_t(w[3] >> 8) << 16));
                    } else {
                        const uint16_t* w = reinterpret_cast<const uint16_t*>(src + 2 + (part & 1) * 8);
                        const uint32_t sh = (part >> 1) * 4;
                        x.x = at_codes4<BF16>(((w[0] >> sh) & 15u) | (((uint32_t(w[0]) >> (8 + sh)) & 15u) << 16));
                        x.y = at_codes4<BF16>(((w[1] >> sh) & 15u) | (((uint32_t(w[1]) >> (8 + sh)) & 15u) << 16));
                        x.z = at_codes4<BF16>(((w[2] >> sh) & 15u) | (((uint32_t(w[2]) >> (8 + sh)) & 15u) << 16));
                        x.w = at_codes4<BF16>(((w[3] >> sh) & 15u) | (((uint32_t(w[3]) >> (8 + sh)) & 15u) << 16));
                    }
                    *reinterpret_cast<uint4*>(dst + at_off<D>(r, c)) = x;
                    if (part == 0) {
                        float d = __half2float(__ushort_as_half(*reinterpret_cast<const uint16_t*>(src)));
                        if (pl && !BF16) {
                            if (fabsf(d) > 65504.f / kAtLift) record_error(P.status, KVM_ERR_NONFINITE, 105);
                            d *= kAtLift;
                        }
                        scales[(pl * 64 + r) * (D / 32) + blk] = d;
                    }
                }
            }
            __syncthreads();
            if (st) compute(t, st, dec, dec + kTile, true);
        }
    }
    if constexpr (QUANT && MODE == kAtTree) {
        // The lifted sums of the quantised pages come down before the tail's are added.
        if (!BF16) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[i][k] *= 1.f / kAtLift;
        }
        // Tail tiles are 16-bit numbers: one at a time through the decoded tile's place.
        for (uint32_t t = max(tb, n_first); t < te; ++t) {
            __syncthreads();
            for (int e = tid; e < kAtKeys * CH; e += kAtThreads) {
                const uint32_t r = e / CH, c = e % CH, x = (t - n_first) * kAtKeys + r;
                const bool valid = x < tail;
                at_cp16(smem_u32(dec) + at_off<D>(r, c), kd + uint64_t(valid ? x : 0) * P.k_tok + c * 16, valid);
                at_cp16(smem_u32(dec) + kTile + at_off<D>(r, c), vd + uint64_t(valid ? x : 0) * P.v_tok + c * 16, valid);
            }
            at_commit();
            at_wait<0>();
            __syncthreads();
            compute(t, state_of(t), dec, dec + kTile, false);
        }
    }
    at_wait<0>();
    grid_release();
    __syncthreads();

    // ---- the warps' parts of each row, merged through shared memory ----
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
        if (qc == 0) sm_ml[wk * M + wm * 16 + qr + 8 * x] = make_float2(mx[x], l[x]);
    }
    __syncthreads();
    constexpr int OS = D + 8;  // floats between rows of the merge buffer
    float* ob = reinterpret_cast<float*>(ring);
    static_assert(size_t(WK) * M * OS * 4 <= size_t(ST) * kStage + (QUANT ? 2 * kTile : 0), "merge buffer");
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int r = wm * 16 + qr + 8 * x;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < WK; ++w) m = fmaxf(m, sm_ml[w * M + r].x);
        const float a = mx[x] == -INFINITY && l[x] == 0.f ? 0.f : fast_exp2(mx[x] - m);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
            *reinterpret_cast<float2*>(ob + (wk * M + r) * OS + i * 8 + qc * 2) =
                make_float2(o[i][2 * x] * a, o[i][2 * x + 1] * a);
    }
    __syncthreads();
    for (int e = tid; e < M * (D / 8); e += kAtThreads) {
        const int r = e / (D / 8), c = e % (D / 8);
        const uint32_t m = m0 + r;
        if (m >= m_end) break;
        float mm = -INFINITY, ll = 0.f;
#pragma unroll
        for (int w = 0; w < WK; ++w) mm = fmaxf(mm, sm_ml[w * M + r].x);
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WK; ++w) {
            const float2 ml = sm_ml[w * M + r];
            if (ml.x != -INFINITY || ml.y != 0.f) ll += ml.y * fast_exp2(ml.x - mm);
            const float4* src = reinterpret_cast<const float4*>(ob + (w * M + r) * OS + c * 8);
            const float4 x = src[0], y = src[1];
            acc[0] += x.x, acc[1] += x.y, acc[2] += x.z, acc[3] += x.w;
            acc[4] += y.x, acc[5] += y.y, acc[6] += y.z, acc[7] += y.w;
        }
        const uint32_t i = m / G, qh = h * G + (m - i * G);
        const uint64_t row_id = (uint64_t(b) * P.width + i) * P.q_heads + qh;
        if (P.splits > 1) {
            const uint64_t id = uint64_t(split) * P.seqs * P.width * P.q_heads + row_id;
            float4* dst = reinterpret_cast<float4*>(P.part_o + id * D + c * 8);
            dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
            dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
            if (c == 0) P.part_ml[id] = make_float2(mm, ll);
        } else {
            const float inv = ll == 0.f ? 0.f : 1.f / ll;
            uint4 w;
            w.x = at_pack<BF16>(acc[0] * inv, acc[1] * inv);
            w.y = at_pack<BF16>(acc[2] * inv, acc[3] * inv);
            w.z = at_pack<BF16>(acc[4] * inv, acc[5] * inv);
            w.w = at_pack<BF16>(acc[6] * inv, acc[7] * inv);
            *reinterpret_cast<uint4*>(P.out + uint64_t(b) * P.o_seq + uint64_t(i) * P.o_row + uint64_t(qh) * P.o_head +
                                      c * 16) = w;
            if (c == 0 && P.lse) P.lse[row_id] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * kAtLn2;
        }
    }
}

// Joins the key chunks of one output row per CTA: rows scaled by 2^(m_c - max m),
// divided by the joined sum. Warps take chunks in turn; chunks that saw nothing
// have a zero sum and are left out.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) attend_combine_kernel(const __grid_constant__ AttendParams P) {
    __shared__ float acc_s[8][D];
    __shared__ float2 ml_s[8];
    grid_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    const uint64_t row_id = blockIdx.x, stride = uint64_t(P.seqs) * P.width * P.q_heads;
    const uint32_t qh = uint32_t(row_id % P.q_heads);
    const uint32_t i = uint32_t((row_id / P.q_heads) % P.width), b = uint32_t(row_id / P.q_heads / P.width);
    const uint32_t rows = P.seq_rows ? __ldg(P.seq_rows + b) : P.width;
    if (i >= rows || rows > P.width) return;
    // A sequence of more rows than the batch has, or than fit its cache, was left out: its partial rows were not
    // written. (A window has no recent tokens and a tree no base: the other's number is 0.)
    const uint64_t base = P.seq_base ? __ldg(reinterpret_cast<const unsigned long long*>(P.seq_base + b)) : P.base;
    const uint32_t recent = P.seq_recent ? __ldg(P.seq_recent + b) : P.recent;
    if (base > P.capacity || rows > P.capacity - base || recent > P.capacity || rows > P.capacity - recent) return;
    // Lane: W neighbouring dims of each 32 * W. Four chunks' loads are started before the first is used.
    constexpr int E = D / 32, W = E < 4 ? E : 4, kAhead = 4;
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    float m = -INFINITY, l = 0.f;
    for (uint32_t c0 = warp; c0 < P.splits; c0 += nw * kAhead) {
        float2 ml[kAhead];
        float x[kAhead][E];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const uint32_t c = c0 + i * nw;
            ml[i] = make_float2(-INFINITY, 0.f);
            if (c < P.splits) {
                ml[i] = P.part_ml[c * stride + row_id];
                const float* src = P.part_o + (c * stride + row_id) * D + lane * W;
#pragma unroll
                for (int e = 0; e < E; e += W) {
                    if constexpr (W == 2) {
                        const float2 v = *reinterpret_cast<const float2*>(src);
                        x[i][0] = v.x, x[i][1] = v.y;
                    } else {
                        const float4 v = *reinterpret_cast<const float4*>(src + e * 32);
                        x[i][e] = v.x, x[i][e + 1] = v.y, x[i][e + 2] = v.z, x[i][e + 3] = v.w;
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (ml[i].y == 0.f) continue;
            const float nm = fmaxf(m, ml[i].x);
            const float a0 = m == -INFINITY ? 0.f : fast_exp2(m - nm), a1 = fast_exp2(ml[i].x - nm);
            m = nm;
            l = l * a0 + ml[i].y * a1;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = acc[e] * a0 + x[i][e] * a1;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) acc_s[warp][(e / W) * 32 * W + lane * W + e % W] = acc[e];
    if (lane == 0) ml_s[warp] = make_float2(m, l);
    __syncthreads();
    float mm = -INFINITY, ll = 0.f;
    for (int w = 0; w < nw; ++w)
        if (ml_s[w].y != 0.f) mm = fmaxf(mm, ml_s[w].x);
    for (int w = 0; w < nw; ++w)
        if (ml_s[w].y != 0.f) ll += ml_s[w].y * fast_exp2(ml_s[w].x - mm);
    const float inv = ll == 0.f ? 0.f : 1.f / ll;
    for (int d = threadIdx.x * 2; d < D; d += blockDim.x * 2) {
        float x = 0.f, y = 0.f;
        for (int w = 0; w < nw; ++w)
            if (ml_s[w].y != 0.f) {
                const float a = fast_exp2(ml_s[w].x - mm);
                x += acc_s[w][d] * a;
                y += acc_s[w][d + 1] * a;
            }
        *reinterpret_cast<uint32_t*>(P.out + uint64_t(b) * P.o_seq + uint64_t(i) * P.o_row + uint64_t(qh) * P.o_head +
                                     d * 2) = at_pack<BF16>(x * inv, y * inv);
    }
    if (threadIdx.x == 0 && P.lse) P.lse[row_id] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * kAtLn2;
}

}  // namespace kvmb
