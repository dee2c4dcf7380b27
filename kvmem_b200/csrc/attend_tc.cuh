// Attention of many rows over a cache on the 5th-generation tensor cores: the
// same operators as attend.cuh (window with sinks, tree over pages), for packed row
// counts where the products and not the reading of K and V bound the time.
//
// One CTA per (sequence, KV head, 128 packed rows, key chunk), in one of two shapes
// (ac_wide): one CTA per SM, or two, so that one's start, end and softmax run beside the
// other's products:
//  * warp 0, in the wide shape also warp 2 (one thread each): TMA loads of 128-key K and V
//    tiles into one ring of 16 KiB units, in the order in which the products take them. A
//    K unit is 128 keys x 64 dims (the B operand of S, K-major); a V unit is 32 / 64 / 128
//    keys x 256 / 128 / 64 dims (the B operand of O, MN-major). Pages come as boxes of
//    gcd(page_tokens, 128) tokens, each from its slot;
//  * warp 1: tcgen05.mma kind::f16, S = Q K^T (M = 128, N = 128, Q in shared memory),
//    then O += P V (N = head_dim, P from tensor memory, where it replaces its S). In
//    the wide shape two S accumulators are in flight (S of tile j + 2 is issued right
//    behind P V of tile j); in the narrow one the tensor core works for the SM's other
//    CTA meanwhile. One commit per product serves the softmax and the ring (a commit
//    costs the tensor core some 100 cycles: with one for each use and unit a tile took
//    4,400 cycles instead of 3,300 at head_dim 256);
//  * softmax warps: thread = packed row = tensor-memory lane; four warps, or eight in the
//    wide shape, each with half of the tile's keys. Masks are words of bits per
//    thread and tile, made only for tiles that some row sees in part. The running max
//    moves lazily: O is rescaled only when it grows by more than 2^8, so P stays
//    below 2^8 and sums stay in 32 bits. P goes to the tensor core in two halves;
//  * warp 3 (and 2): a V tile behind a mask may hold infinities or NaN, which 0 * x
//    would spread to rows that do not see them. Keys that no row sees become zeros; the
//    others are looked through, and where some rows see such a value it is taken out of
//    the product and added by hand to those rows. The tail of a tree waits for its scan, so
//    its sums are four chains and dead keys one bit each (one token over 34 pages of
//    head_dim 256: 33 us before, 24 so); windows keep one chain and a comparison, which
//    leaves the softmax more issue slots (whole prompt 402 us; 411-422 in the tree's form).
// Quantised pages (q8_0 / q4_0): eight more warps read the blocks as stored, decode them to
// fp16 and write them where the copies would have put them. Beside them bf16 queries and keys of
// the tail become fp16, each row after division by a power of two of its own; the tail's values
// stay bf16 (a product of its own type on the same accumulator). A tile of head_dim 256 takes 5.3 us
// of decoding against 1.3 of products and softmax; with four tiles per CTA that is 21 of the 47 us
// below. The rest does not depend on the tiles: the CTA's start, the tail, and 34 chunks to be joined.
//
// Measured (device time at 1,965 MHz, the joining pass included where keys are split):
//   1,024 rows, window 4,096 + 256 sinks, 24 / 4 heads, dim 256, bf16   142 us, 770 TFLOP/s
//   16,381 rows, window 1,000 + 64 sinks, 32 / 8 heads, dim 128, fp16   398 us, 695 TFLOP/s
//     (called for a second and more the GPU's 1,000 W hold it at 1,730 MHz: 447 us, 618 TFLOP/s)
//   60 nodes, 8 lanes, 26 pages of 128, 40 / 8 heads, dim 128, bf16     77 us, 440 TFLOP/s
//   1 node, 34 pages of 256, 24 / 4 heads, dim 256, fp16                25 us, 1.5 TB/s
//   16 nodes, 66 pages of 256, q8_0 / q4_0, 24 / 4 heads, dim 256       47 us (bf16), 40 us (fp16)
//   1 node, the same pages                                              44 us (bf16), 37 us (fp16)
// Every wait is bounded: on expiry the kernel records KVM_ERR_TIMEOUT, raises the
// CTA's abort flag, lets copies and MMAs in flight finish and frees its TMEM.
#pragma once
#include <type_traits>

#include "attend.cuh"
#include "attend_plan.cuh"
#include "prefill_attn.cuh"

namespace kvmb {

constexpr int kAcKeys = 128;             // keys per tile
constexpr uint32_t kAcUnit = 16384;      // bytes per ring unit
constexpr uint32_t kAcTable = 512;       // page boxes of one CTA's key chunk
constexpr uint32_t kAcScans = 8;         // V tiles that the scan's barriers tell apart
constexpr uint32_t kAcMaxTiles = 8;
constexpr uint32_t kAcRaw = 3;           // quantised pages: stages of 32 blocks on their way to a decoding warp
constexpr uint32_t kAcRawBytes = 32 * 34;
constexpr uint32_t kAcScales = 8;        // tail tiles whose key scales are held (K runs at most four tiles ahead of the softmax)

// Two shapes. Wide (head_dim 256): one CTA per SM, two S accumulators, eight softmax
// warps, a deep ring. Narrow (64, 128): two CTAs per SM, each with one S accumulator and
// four softmax warps; the wide shape takes 1.4 times as long there (whole prompt of
// 16,381 rows: 562 us against 397), most of it starts and ends of CTAs in turn.
__host__ __device__ constexpr bool ac_wide(int D) { return D == 256; }
// Quantised pages: the wide shape at every head_dim, with eight more warps that decode.
__host__ __device__ constexpr int ac_threads(int D, bool quant) { return quant ? 640 : ac_wide(D) ? 384 : 256; }
__host__ __device__ constexpr uint32_t ac_units(int D, int mode, bool quant) {
    // What is left of the SM's 227 KiB (or half of it) beside the query tile and the page table.
    return D == 256 ? (quant ? 8u : mode == kAtTree ? 9u : 10u) : D == 128 ? (quant ? 8u : 4u) : (quant ? 6u : 5u);
}
// A K or V tile (D / 64 units) has one full barrier (per half); that of tile q serves tile
// q + ac_tiles again, whose first unit waits for a unit of a tile behind q.
__host__ __device__ constexpr uint32_t ac_tiles(int D, int mode, bool quant) {
    return ac_units(D, mode, quant) / uint32_t(D / 64) + 2u;
}
__host__ __device__ constexpr uint32_t ac_smem_bytes(int D, int mode, bool quant) {
    return 128u * uint32_t(D) * 2u + ac_units(D, mode, quant) * kAcUnit + (ac_wide(D) || quant ? 2048u : 0u) +
           (quant ? 512u + kAcScales * 128u + 8u * kAcRaw * kAcRawBytes : 0u) + (mode == kAtTree ? kAcTable * 8u : 0u) + 544u;
}
static_assert(ac_smem_bytes(256, kAtTree, true) <= 227 * 1024 && ac_smem_bytes(256, kAtWindow, false) <= 227 * 1024, "shared memory");
static_assert(ac_smem_bytes(128, kAtTree, false) <= 113 * 1024 && ac_smem_bytes(64, kAtTree, false) <= 113 * 1024, "shared memory");

struct AttendTcMaps {
    CUtensorMap dk, dv;  // dense keys: (D, kv_heads, tokens, sequences), boxes (64, 1, 128 | V unit keys, 1)
    CUtensorMap pk, pv;  // pages: (D, kv_heads, page_tokens, slots, rows), boxes (64, 1, box | min(box, V unit keys), 1, 1)
};

__device__ __forceinline__ void ac_complete_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

// The instructions of the MMA warp are executed by all its lanes, so that descriptors
// stay in uniform registers; one elected lane issues (the same one every time).
__device__ __forceinline__ void ac_mma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b32 t;\n\telect.sync t|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void ac_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b32 t;\n\telect.sync t|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void ac_commit(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t.reg .b32 t;\n\telect.sync t|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void ac_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
            "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void ac_load_5d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, int v,
                                           uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "r"(smem_u32(bar))
        : "memory");
}

// 0 * x + acc on two packed 16-bit values: stays 0 while every x is finite, NaN from then on.
template <bool BF16>
__device__ __forceinline__ uint32_t ac_zero_times(uint32_t x, uint32_t acc) {
    const uint32_t zero = 0;
    if constexpr (BF16) {
        const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&zero),
                                         *reinterpret_cast<const __nv_bfloat162*>(&acc));
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&zero),
                                  *reinterpret_cast<const __half2*>(&acc));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}

// Words of one block of a quantised row that starts at byte 2 * (odd ? 1 : 0) of its first
// word: {scale, codes}. The last block of a row is an odd one (rows are whole words), so
// its last word ends with the row.
struct AcBlock {
    uint32_t w[9];
    __device__ __forceinline__ void load(const uint8_t* row, uint32_t bi, bool q8) {  // 34 or 18 bytes per block
        const uint32_t* p = reinterpret_cast<const uint32_t*>(row + ((bi * (q8 ? 34u : 18u)) & ~3u));
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = p[i];
        if (q8) {
#pragma unroll
            for (int i = 5; i < 9; ++i) w[i] = p[i];
        }
    }
    __device__ __forceinline__ uint32_t code(int i, bool odd) const { return __funnelshift_rc(w[i], w[i + 1], odd ? 32 : 16); }
    __device__ __forceinline__ uint32_t scale2(bool odd) const {  // the fp16 scale twice
        return __byte_perm(w[0], 0, odd ? 0x3232 : 0x1010);
    }
};

__device__ __forceinline__ uint32_t ac_mul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// 16-byte chunk c (8 values) of a decoded block: code times scale, rounded to fp16 once.
__device__ __forceinline__ uint4 ac_decode_q8(const AcBlock& x, int c, bool odd, uint32_t d2) {
    const uint32_t a = x.code(2 * c, odd), b = x.code(2 * c + 1, odd);
    return make_uint4(ac_mul2(at_codes8<false>(__byte_perm(a, 0, 0x4140)), d2), ac_mul2(at_codes8<false>(__byte_perm(a, 0, 0x4342)), d2),
                      ac_mul2(at_codes8<false>(__byte_perm(b, 0, 0x4140)), d2), ac_mul2(at_codes8<false>(__byte_perm(b, 0, 0x4342)), d2));
}
__device__ __forceinline__ uint4 ac_decode_q4(const AcBlock& x, int c, bool odd, uint32_t d2) {
    const uint32_t sh = (c >> 1) * 4;  // chunks 0, 1: low nibbles of bytes 0-7, 8-15; 2, 3: high nibbles
    const uint32_t a = (x.code(2 * (c & 1), odd) >> sh) & 0x0F0F0F0Fu, b = (x.code(2 * (c & 1) + 1, odd) >> sh) & 0x0F0F0F0Fu;
    return make_uint4(ac_mul2(at_codes4<false>(__byte_perm(a, 0, 0x4140)), d2), ac_mul2(at_codes4<false>(__byte_perm(a, 0, 0x4342)), d2),
                      ac_mul2(at_codes4<false>(__byte_perm(b, 0, 0x4140)), d2), ac_mul2(at_codes4<false>(__byte_perm(b, 0, 0x4342)), d2));
}

// Exponent of the power of two by which a bf16 row is divided before it becomes fp16: it brings the row's largest value
// `top` to [2^13, 2^14). bf16 numbers down to 2^-30 of it are exact then, smaller ones off by at most 2^-38 of it.
__device__ __forceinline__ int ac_row_exponent(float top) {
    const int ex = int((__float_as_uint(top) >> 23) & 255) - 127 - 13;
    return top == 0.f ? 0 : min(max(ex, -120), 114);  // (a NaN or an infinity: the row's products are that anyway)
}
// Whether one of two finite bf16 values lies beyond fp16's largest, 65504: from 65536 on, the next bf16 after 65280
// (the limit that the call sets for a tail beside quantised pages).
__device__ __forceinline__ bool ac_over_half2(uint32_t w) {
    const uint32_t a = w & 0x7FFFu, b = (w >> 16) & 0x7FFFu;
    return (a >= 0x4780u && a < 0x7F80u) || (b >= 0x4780u && b < 0x7F80u);
}

template <int D, bool BF16, int MODE, bool QUANT>
__global__ void __launch_bounds__(ac_threads(D, QUANT), ac_wide(D) || QUANT ? 1 : 2)
    attend_tc_kernel(const __grid_constant__ AttendTcMaps maps, const __grid_constant__ AttendParams P,
                     const uint32_t box) {
    constexpr bool kWide = ac_wide(D) || QUANT;
    constexpr bool OB = BF16 && !QUANT;          // operands of the products in bf16 (decoded pages are fp16)
    // The values of a bf16 tail beside decoded pages stay bf16 (fp16 would lose those below 2^-17), and its P is the sum
    // of two bf16 numbers, 2^-16 of it or less left over: no more is lost than with the fp16 P of the pages.
    constexpr bool kTail16 = BF16 && QUANT;
    constexpr int HS = kWide ? 2 : 1;            // softmax warps per 32 rows
    constexpr uint32_t SB = kWide ? 2 : 1;       // S accumulators
    constexpr uint32_t kScanWarps = kWide ? 1 : 2;
    constexpr int kThreads = ac_threads(D, QUANT);
    constexpr uint32_t kFull = QUANT ? 8 : 1;    // arrivals on a full barrier
    constexpr uint32_t U = D / 64;               // units of a K tile, and of a V tile
    constexpr uint32_t VK = kAcUnit / (D * 2);   // keys of a V unit
    constexpr uint32_t NU = ac_units(D, MODE, QUANT);
    constexpr uint32_t NB = ac_tiles(D, MODE, QUANT);
    static_assert(NB <= kAcMaxTiles && NU >= 2 * U, "ring");
    constexpr uint32_t kQTile = 128 * D * 2;
    constexpr uint32_t kColO = SB * 128, kCols = kWide ? 512 : 256;  // S / P, then O
    extern __shared__ __align__(1024) uint8_t ac_smem[];  // the 128-byte swizzle counts from 1,024-byte boundaries
    uint8_t* qsm = ac_smem;
    uint8_t* ring = qsm + kQTile;
    float* pair_max = reinterpret_cast<float*>(ring + NU * kAcUnit);  // HS = 2: [2 (tile parity)][2 (half)][128]
    float* row_scale = pair_max + (HS == 2 ? 512 : 0);  // QUANT: [128] what the query rows were divided by
    // QUANT, bf16: [kAcScales][128] what the tail's K rows were divided by, 2^(x - 127)
    uint8_t* key_scale = reinterpret_cast<uint8_t*>(row_scale + (QUANT ? 128 : 0));
    uint8_t* raw = key_scale + (QUANT ? kAcScales * 128 : 0);  // QUANT: [8 warps][kAcRaw] blocks
    int2* table = reinterpret_cast<int2*>(raw + (QUANT ? 8 * kAcRaw * kAcRawBytes : 0));
    uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(table) + (MODE == kAtTree ? kAcTable * 8 : 0));
    uint64_t* full = bars;                    // [NB][2] half of the tile's units loaded (its one unit: [0])
    uint64_t* done = full + 2 * kAcMaxTiles;  // [NB] its product is done: S is there (K), O is and P is free (V)
    uint64_t* p_full = done + kAcMaxTiles;  // [2] keys 0 .. 63 of P
    uint64_t* p_half = p_full + 2;          // [2] keys 64 .. 127 of P
    uint64_t* fin = p_full + 4;
    uint64_t* together = p_full + 5;        // all softmax threads (a barrier whose wait is bounded)
    uint64_t* scanned = p_full + 6;         // [kAcScans] V tile looked through
    uint64_t* scaled = scanned + kAcScans;  // [kAcScales] scales of a tail tile's keys are there
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(scaled + kAcScales);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile uint32_t* bad_flag = tmem_slot + 2;  // [kAcScans][2] what the scanning warps found
    static_assert((3 * kAcMaxTiles + 6 + kAcScans + kAcScales) * 8 + 8 + kAcScans * 8 <= 544, "barriers");

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (smem_u32(ac_smem) & 1023u) {
        if (tid == 0) record_error(P.status, KVM_ERR_CUDA, 119);
        return;
    }
    uint32_t un = blockIdx.x;
    const uint32_t mt = un % P.m_tiles;
    un /= P.m_tiles;
    const uint32_t split = un % P.splits;
    un /= P.splits;
    const uint32_t h = un % P.kv_heads, b = un / P.kv_heads;
    const uint32_t G = P.group;
    const uint32_t rows = P.seq_rows ? __ldg(P.seq_rows + b) : P.width;
    if (rows > P.width) {
        if (tid == 0) record_error(P.status, KVM_ERR_LENGTH, 118);
        return;
    }
    const uint32_t m0 = mt * 128, m_end = rows * G;
    if (m0 >= m_end) return;
    auto row_div = [&](uint32_t m) { return uint32_t((uint64_t(m) * P.g_magic) >> P.g_shift); };
    const uint32_t i0 = row_div(m0), i1 = row_div(min(m0 + 127, m_end - 1));

    // ---- this unit's keys (as attend_mma_kernel, tiles of 128) ----
    uint32_t nt, n_first;
    uint32_t p0 = 0, p1 = 0, lo = 0, hi = 0, few = 0;
    uint32_t n_keys = 0, recent = 0, prow = 0;
    const uint32_t bsh = MODE == kAtTree ? 31u - uint32_t(__clz(int(box))) : 0u;  // box = 1 << bsh
    const uint32_t nb = MODE == kAtTree ? uint32_t(kAcKeys) >> bsh : 1;           // boxes of a page tile
    if constexpr (MODE == kAtWindow) {
        const uint64_t base = P.seq_base ? __ldg(reinterpret_cast<const unsigned long long*>(P.seq_base + b)) : P.base;
        if (base > P.capacity || rows > P.capacity - base) {
            if (tid == 0) record_error(P.status, KVM_ERR_LENGTH, 120);
            return;
        }
        p0 = uint32_t(base) + i0;
        p1 = uint32_t(base) + i1;
        hi = p1 + 1;
        lo = P.window == 0 ? hi : (p0 + 1 > P.window ? p0 + 1 - P.window : 0);
        few = min(P.sinks, lo);
        n_first = (few + kAcKeys - 1) / kAcKeys;
        nt = n_first + (hi - lo + kAcKeys - 1) / kAcKeys;
    } else {
        recent = P.seq_recent ? __ldg(P.seq_recent + b) : P.recent;
        if (recent > P.capacity || rows > P.capacity - recent) {
            if (tid == 0) record_error(P.status, KVM_ERR_LENGTH, 121);
            return;
        }
        prow = P.row0 + b * P.row_step;
        uint32_t n_list = P.pool_slots;
        if (P.sel_ids) {
            n_list = __ldg(P.sel_n + b);
            if (n_list > P.sel_width) {
                if (tid == 0) record_error(P.status, KVM_ERR_INVALID_ARGUMENT, 122);
                n_list = P.sel_width;
            }
        }
        n_keys = n_list * P.page_tokens;
        n_first = (n_keys + kAcKeys - 1) / kAcKeys;
        nt = n_first + (recent + rows + kAcKeys - 1) / kAcKeys;
    }
    const uint32_t tb = uint32_t(uint64_t(nt) * split / P.splits), te = uint32_t(uint64_t(nt) * (split + 1) / P.splits);
    const uint32_t n = te - tb;  // tiles of this CTA
    if constexpr (MODE == kAtTree) {
        // The boxes of the chunk's page tiles, so that nobody divides by the page size or looks up a slot later:
        // x = slot, y = first token in the page | (some box of the tile is not full) << 23 | tokens held << 24.
        // The host's chunks have at most kAcTable of them.
        const uint64_t tokens = P.seq_tokens ? __ldg(reinterpret_cast<const unsigned long long*>(P.seq_tokens + b)) : P.tokens;
        const uint32_t page_tiles = tb < n_first ? min(te, n_first) - tb : 0;
        for (uint32_t i = tid; i < min(page_tiles, kAcTable >> (7 - bsh)); i += kThreads) {
            uint32_t least = box;
            for (uint32_t k = 0; k < nb; ++k) {
                const uint32_t x = (tb + i) * kAcKeys + k * box;
                int2 ent = make_int2(0, 0);
                if (x < n_keys) {
                    const uint32_t e = uint32_t((uint64_t(x) * P.pt_magic) >> P.pt_shift), o = x - e * P.page_tokens;
                    int page, slot;
                    if (P.sel_ids) {
                        const uint32_t id = __ldg(P.sel_ids + uint64_t(b) * P.sel_stride + e);
                        page = id < P.pool_pages ? int(id) : -1;
                        slot = page >= 0 ? P.slot_of[uint64_t(prow) * P.pool_pages + page] : -1;
                        if (page < 0) record_error(P.status, KVM_ERR_INVALID_ARGUMENT, 123);
                        else if (slot < 0 || slot >= int(P.pool_slots)) {
                            record_error(P.status, KVM_ERR_STALE, 124);
                            page = -1;
                        }
                    } else {
                        slot = int(e);
                        page = P.page_of[uint64_t(prow) * P.pool_slots + e];
                    }
                    const uint64_t start = uint64_t(max(page, 0)) * P.page_tokens + o;
                    if (page >= 0 && tokens > start) ent = make_int2(slot, int(o | uint32_t(min(tokens - start, uint64_t(box))) << 24));
                }
                least = min(least, uint32_t(ent.y) >> 24);
                table[i * nb + k] = ent;
            }
            if (least < box) table[i * nb].y |= 1 << 23;
        }
    }

    if (tid == 0) {
        for (uint32_t i = 0; i < NB; ++i) {
            mbar_init(&full[2 * i], kFull);
            mbar_init(&full[2 * i + 1], kFull);
            mbar_init(&done[i], 1);
        }
        for (uint32_t i = 0; i < kAcScans; ++i) mbar_init(&scanned[i], kScanWarps);
        if (QUANT)
            for (uint32_t i = 0; i < kAcScales; ++i) mbar_init(&scaled[i], 8);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&p_full[i], 128);
            mbar_init(&p_half[i], 128);
        }
        mbar_init(fin, 1);
        mbar_init(together, 128 * HS);
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp >= 4 && warp < 4 + 4 * HS) {
        // The query tile, a row by D / 8 lanes.
        constexpr uint32_t kLanes = D / 8, kRows = 128 * HS / kLanes, kIts = 128 / kRows;  // rows at a time; rounds
        constexpr uint32_t kBatch = kIts < 8 ? kIts : 8;                                   // loads in flight
        const uint32_t base_row = uint32_t(tid - 128) / kLanes, c = uint32_t(tid) % kLanes;
        uint8_t* qd = qsm + (c >> 3) * 16384;
#pragma unroll
        for (uint32_t it = 0; it < kIts; it += kBatch) {
            uint4 x[kBatch];
#pragma unroll
            for (uint32_t k = 0; k < kBatch; ++k) {
                const uint32_t r = min(m0 + base_row + (it + k) * kRows, m_end - 1), i = row_div(r);
                x[k] = __ldg(reinterpret_cast<const uint4*>(P.q + uint64_t(b) * P.q_seq + uint64_t(i) * P.q_row +
                                                            uint64_t(h * G + (r - i * G)) * P.q_head) + c);
            }
#pragma unroll
            for (uint32_t k = 0; k < kBatch; ++k) {
                // (rows past the last hold copies of it: computed and not written)
                const uint32_t row = base_row + (it + k) * kRows;
                if constexpr (QUANT && BF16) {
                    // As fp16, divided by a power of two.
                    float v[8], top = 0.f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t w = e == 0 ? x[k].x : e == 1 ? x[k].y : e == 2 ? x[k].z : x[k].w;
                        const float2 f = at_unpack<BF16>(w);
                        v[2 * e] = f.x, v[2 * e + 1] = f.y;
                        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
#pragma unroll
                    for (uint32_t o = kLanes / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    const int ex = ac_row_exponent(top);
                    const float inv = __uint_as_float(uint32_t(127 - ex) << 23);
                    __half2 hv[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) hv[e] = __floats2half2_rn(v[2 * e] * inv, v[2 * e + 1] * inv);
                    x[k] = *reinterpret_cast<uint4*>(hv);
                    if (c == 0) row_scale[row] = __uint_as_float(uint32_t(127 + ex) << 23);
                }
                *reinterpret_cast<uint4*>(qd + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = x[k];
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tc_fence_before();
    // The K loads need the barriers alone, which their own thread has set up (and the page
    // table): over a dense cache they start at once.
    if (MODE == kAtWindow && warp == 0) {
        __threadfence_block();
        asm volatile("bar.arrive 1, %0;" ::"n"(kThreads) : "memory");
    } else {
        named_sync(1, kThreads);
    }
    tc_fence_after();
    const uint32_t tmem = warp ? *tmem_slot : 0;

    // Ring order of the tiles, the order in which the products take them.
    // One S: K0 V0 K1 V1 ..; two: K0 K1 V0 K2 V1 .. V(n - 1).
    auto k_seq = [&](uint32_t j) { return SB == 1 ? 2 * j : (j ? 2 * j - 1 : 0); };
    auto v_seq = [&](uint32_t j) { return SB == 1 ? 2 * j + 1 : (j + 1 == n ? 2 * n - 1 : 2 * j + 2); };
    // The q-th tile of the ring (SB = 2): K or V, and which.
    [[maybe_unused]] auto ring_v = [&](uint32_t q) { return q + 1 == 2 * n || (q && !(q & 1)); };
    [[maybe_unused]] auto ring_tile = [&](uint32_t q) { return q + 1 == 2 * n ? n - 1 : ring_v(q) ? q / 2 - 1 : (q + 1) / 2; };
    // Whether some row of the CTA does not see all of tile t.
    auto in_part = [&](uint32_t t) -> bool {
        if constexpr (MODE == kAtWindow) {
            const uint32_t a = t < n_first ? t * kAcKeys : lo + (t - n_first) * kAcKeys;
            return !(a + kAcKeys <= (t < n_first ? few : hi) && a + kAcKeys - 1 <= p0 &&
                     (a + kAcKeys <= P.sinks || p1 - a < P.window));
        } else {
            if (t >= n_first) return (t - n_first + 1) * kAcKeys > recent;
            return (table[(t - tb) * nb].y >> 23) & 1;
        }
    };

    // Two CTAs per SM: registers go to the softmax warps, 4 x 32 x 72 + 4 x 32 x 184 = 256 x 128.
    // With decoding warps: 4 x 32 x 64 + 8 x 32 x 136 + 8 x 32 x 72 = 640 x 96.
    if (warp < 4) {
        if constexpr (QUANT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kAcQuantIssue));
        else if constexpr (HS == 1) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kAcNarrowIssue));
        if (QUANT && (warp == 0 || warp == 2)) {
            // (the decoding warps fill the ring)
        } else if (warp == 0 || (kScanWarps == 1 && warp == 2)) {
            // ---- TMA producer; in the wide shape two, warp 0 for K and warp 2 for V (one thread's 20 copies
            // per tile of head_dim 256 took 2,600 cycles to issue, more than the tile's products) ----
            if (lane == 0) {
                uint32_t freed = 0;  // tiles known to be used up
                // K (or V) tile j of this CTA, the q-th of the ring.
                auto load = [&](uint32_t j, auto v) -> bool {
                    constexpr bool kV = decltype(v)::value;
                    constexpr uint32_t kKeys = kV ? VK : uint32_t(kAcKeys), kBlocks = kV ? U : 1;  // keys, 64-dim blocks of a unit
                    constexpr uint32_t kPer = U > 1 ? U / 2 : 1;                                   // units per barrier
                    const CUtensorMap* dmap = kV ? &maps.dv : &maps.dk;
                    const CUtensorMap* pmap = kV ? &maps.pv : &maps.pk;
                    const uint32_t q = kV ? v_seq(j) : k_seq(j), t = tb + j, bh = min(box, kKeys);
                    const bool dense = MODE == kAtWindow || t >= n_first;
                    const uint32_t tok = MODE == kAtWindow ? (t < n_first ? t * kAcKeys : lo + (t - n_first) * kAcKeys)
                                                           : (t - n_first) * kAcKeys;
                    const int2* ents = table + j * nb;  // (page tiles come first: tile j of this CTA is tile tb + j)
                    uint64_t* bar = nullptr;
                    uint32_t left = 0;  // bytes of the barrier's copies that are not started
#pragma unroll
                    for (uint32_t sub = 0; sub < U; ++sub) {
                        const uint32_t idx = q * U + sub, s = idx % NU;
                        while (idx >= NU && freed <= (idx - NU) / U) {  // the tile whose unit this one replaces
                            if (!mbar_wait(&done[freed % NB], (freed / NB) & 1)) {
                                record_error(P.status, KVM_ERR_TIMEOUT, 125);
                                if (left) ac_complete_tx(bar, left);
                                return false;
                            }
                            ++freed;
                        }
                        if (sub % kPer == 0) {
                            bar = &full[(q % NB) * 2 + sub / kPer];
                            left = kPer * kAcUnit;
                            mbar_arrive_expect_tx(bar, left);
                        }
                        left -= kAcUnit;
                        const uint32_t dst = smem_u32(ring + s * kAcUnit), key0 = kV ? sub * VK : 0;
                        if (dense) {
#pragma unroll
                            for (uint32_t a = 0; a < kBlocks; ++a)
                                ac_load_4d(dst + a * kKeys * 128, dmap, int((kV ? a : sub) * 64), int(h), int(tok + key0), int(b), bar);
                        } else {
                            for (uint32_t i = 0; i < kKeys; i += bh) {
                                const int2 ent = ents[(key0 + i) >> bsh];
                                const uint32_t in = (key0 + i) & (box - 1);
                                // A box without a token is read past the last slot: zeros.
                                const int slot = in < uint32_t(ent.y) >> 24 ? ent.x : int(P.pool_slots);
#pragma unroll
                                for (uint32_t a = 0; a < kBlocks; ++a)
                                    ac_load_5d(dst + a * kKeys * 128 + i * 128, pmap, int((kV ? a : sub) * 64), int(h),
                                               int((uint32_t(ent.y) & 0x7FFFFFu) + in), slot, int(prow), bar);
                            }
                        }
                    }
                    return true;
                };
                // V(j) stays at most two tiles ahead of the scan (below).
                auto load_v = [&](uint32_t j) -> bool {
                    if (j >= 2 && !mbar_wait(&scanned[(j - 2) % kAcScans], ((j - 2) / kAcScans) & 1)) {
                        record_error(P.status, KVM_ERR_TIMEOUT, 127);
                        return false;
                    }
                    return load(j, std::true_type{});
                };
                bool ok = true;
                uint32_t j = 0;
                if (kScanWarps == 2) {
                    if (n) ok = load(0, std::false_type{});
                    for (; j < n && ok && !*abort_flag; ++j) ok = load_v(j) && (j + 1 >= n || load(j + 1, std::false_type{}));
                } else if (warp == 0) {
                    for (; j < n && ok && !*abort_flag; ++j) ok = load(j, std::false_type{});
                } else {
                    for (; j < n && ok && !*abort_flag; ++j) ok = load_v(j);
                }
                if (!ok) *abort_flag = 1;
                // Every issued copy lands before the CTA frees its shared memory: the tiles whose barrier has
                // not been taken over by a later one (which its release came before).
                for (uint32_t i = j > NB ? j - NB : 0; i < j; ++i)
                    for (uint32_t v = kScanWarps == 2 ? 0 : warp / 2; v <= (kScanWarps == 2 ? 1u : uint32_t(warp) / 2); ++v) {
                        const uint32_t q = v ? v_seq(i) : k_seq(i);
                        if (ok ? q + NB < 2 * n : q < freed) continue;
                        for (uint32_t x = 0; x < (U > 1 ? 2u : 1u); ++x)
                            if (!mbar_wait(&full[(q % NB) * 2 + x], (q / NB) & 1)) record_error(P.status, KVM_ERR_TIMEOUT, 126);
                    }
            }
        } else if (warp == 1) {
            // ---- MMA issue: tile j, S accumulator j % SB ----
            // The warp only adds constants to descriptors and ring positions.
            constexpr uint32_t idesc_s = pf_idesc(128, kAcKeys, OB, false);
            constexpr uint32_t idesc_o = pf_idesc(128, D, OB, true), idesc_tail = pf_idesc(128, D, true, true);
            const uint32_t page_steps = kTail16 ? __shfl_sync(0xffffffffu, tb < n_first ? n_first - tb : 0, 0) : 0;
            const uint64_t qdesc = tc_desc_sw128(smem_u32(qsm)), kdesc = tc_desc_sw128(smem_u32(ring));
            const uint64_t vdesc = pf_desc_mn_sw128(smem_u32(ring), VK * 128);
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), steps = __shfl_sync(0xffffffffu, n, 0);
            struct Pos {  // a unit of the ring; a tile's barrier and the parity of its pass
                uint32_t s, b, ph;
                __device__ __forceinline__ void unit() { s = s + 1 == NU ? 0 : s + 1; }
                __device__ __forceinline__ void tile() {
                    if (++b == NB) b = 0, ph ^= 1;
                }
                __device__ __forceinline__ void skip() {  // a whole tile
                    s += U;
                    if (s >= NU) s -= NU;
                    tile();
                }
            };
            Pos kp{0, 0, 0}, vp{0, 0, 0};
            vp.skip();
            if (SB == 2 && steps > 1) vp.skip();
            int err = 0;
            // S from the K tile at kp, which moves on (over the V tile in between, but for K1 of two).
            auto issue_s = [&](uint32_t slot, bool over) -> bool {
#pragma unroll
                for (uint32_t a = 0; a < U; ++a) {
                    if (a == 0 || a == U / 2) {
                        if (!pf_warp_wait(&full[kp.b * 2 + (a ? 1 : 0)], kp.ph)) return false;
                        // Decoded K comes in halves of keys, loaded K in halves of dims.
                        if (QUANT && U > 1 && a == 0 && !pf_warp_wait(&full[kp.b * 2 + 1], kp.ph)) return false;
                        tc_fence_after();
                    }
                    const uint64_t kd = kdesc + kp.s * (kAcUnit >> 4);
#pragma unroll
                    for (uint32_t kk = 0; kk < 4; ++kk)
                        ac_mma(tm + slot * 128, qdesc + a * (16384 >> 4) + kk * 2, kd + kk * 2, idesc_s, (a | kk) != 0);
                    kp.unit();
                }
                ac_commit(&done[kp.b]);
                kp.tile();
                if (over) kp.skip();
                return true;
            };
            for (uint32_t j = 0; j < SB && j < steps && !err; ++j)
                if (!issue_s(j, SB == 1 || j > 0)) err = 131;
            for (uint32_t j = 0; j < steps && !err; ++j) {
                const uint32_t slot = j % SB, ph = (j / SB) & 1;
                if (!pf_warp_wait(&full[vp.b * 2], vp.ph)) err = 133;
                if (!err && !pf_warp_wait(&p_full[slot], ph)) err = 132;
                if (err || __shfl_sync(0xffffffffu, *abort_flag, 0)) {
                    if (!err) err = -1;
                    break;
                }
                tc_fence_after();
#pragma unroll
                for (uint32_t a = 0; a < U; ++a) {
                    if (U > 1 && a == U / 2 && !pf_warp_wait(&full[vp.b * 2 + 1], vp.ph)) err = 133;
                    const uint64_t vd = vdesc + vp.s * (kAcUnit >> 4);
#pragma unroll
                    for (uint32_t kk = 0; kk < VK / 16; ++kk) {  // P: 16 keys = 8 tensor-memory columns
                        if (a * VK + kk * 16 == 64) {
                            if (!pf_warp_wait(&p_half[slot], ph)) err = 136;
                            tc_fence_after();
                        }
                        const bool tail = kTail16 && j >= page_steps;
                        ac_mma_ts(tm + kColO, tm + slot * 128 + (a * (VK / 16) + kk) * 8, vd + kk * (2048 >> 4),
                                  tail ? idesc_tail : idesc_o, j > 0 || (a | kk) != 0);
                        if (tail)
                            ac_mma_ts(tm + kColO, tm + slot * 128 + 64 + (a * (VK / 16) + kk) * 8, vd + kk * (2048 >> 4), idesc_tail, 1);
                    }
                    vp.unit();
                }
                ac_commit(&done[vp.b]);
                vp.tile();
                // Over the K tile in between; of two S none stands before the last V tile.
                if (SB == 1 || j + 2 < steps) vp.skip();
                if (!err && j + SB < steps && !issue_s(slot, true)) err = 131;
            }
            if (err > 0 && lane == 0) {
                record_error(P.status, KVM_ERR_TIMEOUT, err);
                *abort_flag = 1;
            }
            __syncwarp();
            ac_commit(fin);
            if (!pf_warp_wait(fin, 0) && lane == 0) record_error(P.status, KVM_ERR_TIMEOUT, 134);
        } else {
            // ---- V tiles that some row does not see in full are looked through ----
            // (It waits for every V tile, and the V loads stay at most two tiles ahead of it: were it to
            // look at a barrier of another pass, that pass's parity could be taken for its tile's.)
            for (uint32_t j = 0; j < n; ++j) {
                const uint32_t q = v_seq(j);
                bool ok = pf_warp_wait(&full[(q % NB) * 2], (q / NB) & 1);
                if (U > 1) ok = pf_warp_wait(&full[(q % NB) * 2 + 1], (q / NB) & 1) && ok;
                const uint32_t t = tb + j;
                bool found = false;
                auto scan = [&](auto as_bf16) {  // (in the type of the tile's values)
                    constexpr bool B = decltype(as_bf16)::value;
                    uint32_t acc[4] = {};
                    // V rows of keys that no row sees become zeros; the others are looked through.
                    [[maybe_unused]] const bool paged = MODE == kAtTree && t < n_first;
                    const uint32_t live = MODE == kAtWindow ? (t < n_first ? few - t * kAcKeys : hi - lo - (t - n_first) * kAcKeys)
                                                            : recent + rows - (t - n_first) * kAcKeys;
                    constexpr uint32_t kStep = 32 * kScanWarps;
                    const uint32_t first = uint32_t(tid - (128 - 32 * int(kScanWarps)));
                    uint32_t dead[4] = {};  // a bit per key (pages)
                    if constexpr (MODE == kAtTree) {
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) {
                            const uint32_t key = i * 32 + lane;
                            dead[i] = __ballot_sync(0xffffffffu, paged ? (key & (box - 1)) >= uint32_t(table[j * nb + (key >> bsh)].y) >> 24
                                                                       : key >= live);
                        }
                    }
                    [[maybe_unused]] const bool some = dead[0] | dead[1] | dead[2] | dead[3];
                    for (uint32_t a = 0; a < U; ++a) {
                        uint4* v4 = reinterpret_cast<uint4*>(ring + ((q * U + a) % NU) * kAcUnit) + first;
                        for (uint32_t e0 = 0; e0 < kAcUnit / 16; e0 += 8 * kStep) {
                            uint4 y[8];
#pragma unroll
                            for (uint32_t i = 0; i < 8; ++i) y[i] = v4[e0 + i * kStep];
#pragma unroll
                            for (uint32_t i = 0; i < 8; ++i) {
                                const uint32_t key = a * VK + ((e0 + i * kStep + first) / 8) % VK;
                                if constexpr (MODE == kAtWindow) {
                                    if (key >= live) v4[e0 + i * kStep] = make_uint4(0, 0, 0, 0);
                                    else acc[0] = ac_zero_times<B>(y[i].x, ac_zero_times<B>(y[i].y, ac_zero_times<B>(y[i].z, ac_zero_times<B>(y[i].w, acc[0]))));
                                } else {
                                    const uint32_t lo2 = key & 32 ? dead[1] : dead[0], hi2 = key & 32 ? dead[3] : dead[2];
                                    if (some && (((key & 64 ? hi2 : lo2) >> (key & 31)) & 1)) v4[e0 + i * kStep] = y[i] = make_uint4(0, 0, 0, 0);
                                    acc[0] = ac_zero_times<B>(y[i].x, acc[0]), acc[1] = ac_zero_times<B>(y[i].y, acc[1]);
                                    acc[2] = ac_zero_times<B>(y[i].z, acc[2]), acc[3] = ac_zero_times<B>(y[i].w, acc[3]);
                                }
                            }
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    found = at_nonfinite<B>(acc[0]) || at_nonfinite<B>(acc[1]) || at_nonfinite<B>(acc[2]) || at_nonfinite<B>(acc[3]);
                };
                if (in_part(t)) {
                    if (kTail16 && t >= n_first) scan(std::true_type{});
                    else scan(std::bool_constant<OB>{});
                }
                const bool bad = __any_sync(0xffffffffu, found);
                if (lane == 0) {
                    bad_flag[(j % kAcScans) * 2 + (warp & 1)] = bad;
                    mbar_arrive(&scanned[j % kAcScans]);
                }
                if (!ok || __shfl_sync(0xffffffffu, *abort_flag, 0)) break;
            }
        }
    } else if (QUANT && warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kAcQuantDecode));
        // ---- decoding warps: K and V tiles in ring order, 256 threads per tile ----
        // Each warp brings the rows of 32 blocks at a time into stages of its own (16, 8 or 4 bytes per copy,
        // as the rows' sizes and strides allow; a thread's loads of its own block touch 8 or more lines per
        // word, and with them a tile of head_dim 256 took 12,400 cycles), then one thread decodes
        // one block: code times scale in fp16, each product rounded once, half a step of fp16, 2^-11;
        // reported where a scale above 511 could leave its range. Keys without a token become zeros.
        const uint32_t dw = uint32_t(warp) - 12, dt = uint32_t(tid) - 384;
        constexpr uint32_t kBlk = D / 32, kWarpKeys = 32 / kBlk, kKeys = 8 * kWarpKeys, kHalves = U > 1 ? 2 : 1;
        uint32_t freed = 0;
        bool ok = true, wild = false;
        // 16-byte chunk c (of the row's D / 8) of key `key` of the tile whose first unit is `at`.
        auto place = [&](uint32_t at, bool v, uint32_t key, uint32_t c) -> uint4* {
            const uint32_t u = v ? key / VK : c >> 3, r = v ? key % VK : key;
            return reinterpret_cast<uint4*>(ring + ((at + u) % NU) * kAcUnit + (v ? (c >> 3) * VK * 128 : 0u) + r * 128 +
                                            (((c & 7) ^ (r & 7)) << 4));
        };
        auto done_half = [&](uint32_t q, uint32_t hf) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[(q % NB) * 2 + hf]);
        };
        const bool kq8 = P.pk_type == KVM_Q8_0, vq8 = P.pv_type == KVM_Q8_0;
        // This thread's key (of a stage) and block: the stores of eight lanes fall on the eight chunks of the
        // swizzle (eight keys, or four keys and a pair of blocks).
        const uint32_t mine = kBlk == 8 ? lane & 3u : (uint32_t(lane) >> 3) / kBlk * 8 + (lane & 7u);
        const uint32_t bi = kBlk == 8 ? uint32_t(lane) >> 2 : (uint32_t(lane) >> 3) % kBlk;
        const bool odd = bi & 1;
        const uint8_t* kbase = P.pk + uint64_t(prow) * P.pk_row + uint64_t(h) * P.pk_head;
        const uint8_t* vbase = P.pv + uint64_t(prow) * P.pv_row + uint64_t(h) * P.pv_head;
        uint8_t* stage = raw + dw * kAcRaw * kAcRawBytes;
        // The warp's keys of a stage lie in one box (boxes hold 16 tokens or more): {slot, first token | tokens << 24}.
        auto entry = [&](const int2* ents, uint32_t k0) {
            const uint32_t key = k0 + dw * kWarpKeys;
            int2 e = ents[key >> bsh];
            const uint32_t in = key & (box - 1), held = uint32_t(e.y) >> 24;
            e.y = int((uint32_t(e.y) & 0x7FFFFFu) + in | (held > in ? min(held - in, kWarpKeys) : 0u) << 24);
            return e;
        };
        // Next stage to copy: ring position, key, buffer; and what its tile's stages share.
        uint32_t cq = 0, ck = 0, cs = 0, c_gran = 0;
        const int2* c_ents = table;
        const uint8_t* c_base = nullptr;
        uint64_t c_slot = 0, c_tok = 0;
        bool c_q8 = false;
        auto copy = [&]() {
            if (ck == 0) {
                while (cq < 2 * n && tb + ring_tile(cq) >= n_first) ++cq;
                const bool v = ring_v(cq);
                c_ents = table + ring_tile(cq) * nb;
                c_base = v ? vbase : kbase, c_slot = v ? P.pv_slot : P.pk_slot, c_tok = v ? P.pv_tok : P.pk_tok;
                c_gran = v ? P.pv_gran : P.pk_gran, c_q8 = v ? vq8 : kq8;
            }
            if (cq < 2 * n) {
                const int2 e = entry(c_ents, ck);
                const uint64_t tok_bytes = c_tok;
                const uint8_t* src = c_base + uint64_t(uint32_t(e.x)) * c_slot + uint64_t(uint32_t(e.y) & 0xFFFFFFu) * tok_bytes;
                const uint32_t gran = c_gran;
                const uint32_t some = uint32_t(e.y) >> 24, dst = smem_u32(stage + cs * kAcRawBytes);
                auto rows_of = [&](auto g, auto bytes) {
                    constexpr uint32_t kG = decltype(g)::value, kPer = kBlk * decltype(bytes)::value / kG;
#pragma unroll
                    for (uint32_t i0 = 0; i0 < kWarpKeys * kPer; i0 += 32) {
                        const uint32_t i = i0 + lane, r = i / kPer, o = (i - r * kPer) * kG;
                        if (r >= some) continue;
                        const uint8_t* from = src + r * tok_bytes + o;
                        if constexpr (kG == 16) at_cp16(dst + i * kG, from, true);
                        else if constexpr (kG == 8) at_cp8(dst + i * kG, from, true);
                        else at_cp4(dst + i * kG, from, true);
                    }
                };
                auto plane = [&](auto bytes) {
                    if constexpr (kBlk * decltype(bytes)::value % 16 == 0) {
                        if (gran == 16) return rows_of(std::integral_constant<uint32_t, 16>{}, bytes);
                    }
                    if constexpr (kBlk * decltype(bytes)::value % 8 == 0) {
                        if (gran >= 8) return rows_of(std::integral_constant<uint32_t, 8>{}, bytes);
                    }
                    rows_of(std::integral_constant<uint32_t, 4>{}, bytes);
                };
                if (c_q8) plane(std::integral_constant<uint32_t, 34>{});
                else plane(std::integral_constant<uint32_t, 18>{});
                cs = cs + 1 == kAcRaw ? 0 : cs + 1;
                ck += kKeys;
                if (ck == uint32_t(kAcKeys)) ck = 0, ++cq;
            }
            at_commit();
        };
#pragma unroll 1
        for (uint32_t i = 0; i < kAcRaw; ++i) copy();
        uint32_t rs = 0;  // the buffer to read next
        AcBlock x;
        for (uint32_t q = 0; q < 2 * n && ok; ++q) {
            const bool v = ring_v(q);
            const uint32_t j = ring_tile(q), t = tb + j, at = q * U, last = at + U - 1;
            while (ok && last >= NU && freed <= (last - NU) / U) {  // the tiles whose units this one replaces
                ok = pf_warp_wait(&done[freed % NB], (freed / NB) & 1);
                ++freed;
            }
            if (ok && v && j >= 2) ok = pf_warp_wait(&scanned[(j - 2) % kAcScans], ((j - 2) / kAcScans) & 1);
            if (!ok || __shfl_sync(0xffffffffu, *abort_flag, 0)) break;
            if (t < n_first) {
                for (uint32_t k0 = 0; k0 < uint32_t(kAcKeys) && ok; k0 += kKeys) {
                    at_wait<kAcRaw - 1>();
                    __syncwarp();
                    x.load(stage + rs * kAcRawBytes + mine * (v ? P.pv_bytes : P.pk_bytes), bi, v ? vq8 : kq8);
                    rs = rs + 1 == kAcRaw ? 0 : rs + 1;
                    const bool live = mine < uint32_t(entry(table + j * nb, k0).y) >> 24;
                    __syncwarp();
                    copy();
                    const uint32_t key = k0 + dw * kWarpKeys + mine, d2 = live ? x.scale2(odd) : 0u;
                    wild = wild || (d2 & 0x7FFFu) > 0x5FFCu;  // 511
                    // (a dead key's bytes are whatever the stage held; its scale is zero)
                    uint4* to[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) to[c] = place(at, v, key, bi * 4 + c);
                    auto put = [&](auto as_q8) {
                        uint4 z[4];
#pragma unroll
                        for (int c = 0; c < 4; ++c) z[c] = decltype(as_q8)::value ? ac_decode_q8(x, c, odd, d2) : ac_decode_q4(x, c, odd, d2);
#pragma unroll
                        for (int c = 0; c < 4; ++c) *to[c] = z[c];
                    };
                    if (v ? vq8 : kq8) put(std::true_type{});
                    else put(std::false_type{});
                    if ((k0 + kKeys) % (kAcKeys / kHalves) == 0) done_half(q, (k0 + kKeys) / (kAcKeys / kHalves) - 1);
                }
            } else {
                // The tail's 16-bit rows.
                const uint32_t tok0 = (t - n_first) * kAcKeys, most = recent + rows;
                // A row by kCh lanes; kBatch rows' loads are started before the first is used.
                constexpr uint32_t kCh = D / 8, kIts = 128 * kCh / 256, kBatch = kIts < 8 ? kIts : 8;
                const uint32_t c = uint32_t(lane) % kCh;
                const uint8_t* head = v ? P.v + uint64_t(b) * P.v_seq + uint64_t(h) * P.v_head : P.k + uint64_t(b) * P.k_seq + uint64_t(h) * P.k_head;
                const uint64_t tok_bytes = v ? P.v_tok : P.k_tok;
#pragma unroll 1
                for (uint32_t i0 = 0; i0 < kIts; i0 += kBatch) {
                    uint4 z[kBatch];
                    const uint32_t key0 = (dt + i0 * 256) / kCh;
#pragma unroll
                    for (uint32_t k = 0; k < kBatch; ++k) {
                        const uint32_t key = key0 + k * (256 / kCh);
                        z[k] = make_uint4(0, 0, 0, 0);
                        if (tok0 + key < most) z[k] = __ldg(reinterpret_cast<const uint4*>(head + uint64_t(tok0 + key) * tok_bytes) + c);
                    }
#pragma unroll
                    for (uint32_t k = 0; k < kBatch; ++k) {
                        const uint32_t key = key0 + k * (256 / kCh);
                        if constexpr (BF16) {
                            wild = wild || ac_over_half2(z[k].x) || ac_over_half2(z[k].y) || ac_over_half2(z[k].z) || ac_over_half2(z[k].w);
                            if (!v) {  // K rows as fp16, divided by a power of two as the query rows are
                                constexpr uint32_t kAbs = 0x7FFF7FFFu;
                                uint32_t m = __vmaxu2(__vmaxu2(z[k].x & kAbs, z[k].y & kAbs), __vmaxu2(z[k].z & kAbs, z[k].w & kAbs));
#pragma unroll
                                for (uint32_t o = kCh / 2; o; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
                                const int ex = ac_row_exponent(__uint_as_float(max(m & 0xFFFFu, m >> 16) << 16));
                                const float inv = __uint_as_float(uint32_t(127 - ex) << 23);
                                auto scaled2 = [&](uint32_t w) {
                                    const float2 f = at_unpack<BF16>(w);
                                    return pf_pack2<false>(f.x * inv, f.y * inv);
                                };
                                z[k] = make_uint4(scaled2(z[k].x), scaled2(z[k].y), scaled2(z[k].z), scaled2(z[k].w));
                                if (c == 0) key_scale[((t - max(tb, n_first)) % kAcScales) * 128 + key] = uint8_t(127 + ex);
                            }
                        }
                        *place(at, v, key, c) = z[k];
                    }
                }
                if (kTail16 && !v) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&scaled[(t - max(tb, n_first)) % kAcScales]);
                }
                for (uint32_t hf = 0; hf < kHalves; ++hf) done_half(q, hf);
            }
        }
        at_wait<0>();
        if (wild) record_error(P.status, KVM_ERR_NONFINITE, 128);
        if (!ok && lane == 0) {
            record_error(P.status, KVM_ERR_TIMEOUT, 129);
            *abort_flag = 1;
        }
    } else {
        if constexpr (QUANT) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kAcQuantSoftmax));
        else if constexpr (HS == 1) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kAcNarrowSoftmax));
        // ---- softmax: thread = packed row (tensor-memory lane), NK of the tile's keys ----
        // With two warps per 32 rows these exchange their maxes through shared memory, behind a
        // barrier of their own. A warp that gives up raises the abort flag and then arrives there,
        // and its partner looks at the flag behind every such barrier: no wait stays open.
        constexpr int NK = kAcKeys / HS, NW = NK / 32;
        const uint32_t half = HS == 2 ? uint32_t(tid - 128) / 128 : 0u, row = uint32_t(tid) & 127;
        const uint32_t lane_addr = tmem + ((32u * uint32_t(warp & 3)) << 16);
        const uint32_t r = m0 + row;  // packed row
        const uint32_t ri = row_div(min(r, m_end - 1));
        const uint32_t qh = h * G + (min(r, m_end - 1) - ri * G);
        const uint32_t pair = 2 + uint32_t(warp & 3);  // barrier
        float* xch = pair_max + row;
        const float c2 = QUANT && BF16 ? P.scale_log2 * row_scale[row] : P.scale_log2;
        float m_used = -1e30f, l = 0.f;
        bool ok = true;
        uint32_t meet_phase = 0;
        auto meet = [&] {
            mbar_arrive(together);
            ok = pf_warp_wait(together, meet_phase) && ok;
            meet_phase ^= 1;
        };
        auto pair_sync = [&] {
            if constexpr (HS == 2) named_sync(pair, 64);
            ok = ok && !__shfl_sync(0xffffffffu, *abort_flag, 0);
        };
        auto below = [](int x, int q4) -> uint32_t {  // bits of the keys < x in word q4
            const int y = min(max(x - q4 * 32, 0), 32);
            return y == 32 ? ~0u : (1u << y) - 1u;
        };
        const uint32_t col_o = lane_addr + kColO + half * (D / HS);  // this thread's part of the row's O
        for (uint32_t j = 0; j < n; ++j) {
            const uint32_t slot = j % SB, t = tb + j;
            // Which of its keys this row sees; `part`: some row of the CTA does not see all of the tile.
            uint32_t see[NW];
#pragma unroll
            for (int q = 0; q < NW; ++q) see[q] = ~0u;
            const bool part = in_part(t);
            if (part) {
                if (MODE == kAtWindow) {
                    // Keys [0, s1) u [w0, u1) of the tile: sinks, and the window up to the row's position.
                    const uint32_t a = t < n_first ? t * kAcKeys : lo + (t - n_first) * kAcKeys;
                    const uint32_t end = t < n_first ? few : hi, p = p0 + (ri - i0);
                    const int u1 = int(min(end, p + 1)) - int(a);
                    const int s1 = min(P.sinks > a ? int(min(P.sinks - a, 256u)) : 0, u1);
                    const int w0 = P.window == 0 ? 256 : (p + 1 > P.window ? int(p + 1 - P.window) - int(a) : 0);
#pragma unroll
                    for (int q = 0; q < NW; ++q) {
                        const int q4 = int(half) * NW + q;
                        see[q] = below(s1, q4) | (below(u1, q4) & ~below(w0, q4));
                    }
                } else if (t >= n_first) {
                    const int rec = int(recent) - int((t - n_first) * kAcKeys);  // keys below are recent tokens, key rec + x is node x
                    const uint32_t* tw = P.tree ? P.tree + uint64_t(b) * P.tree_seq + uint64_t(ri) * P.tree_words : nullptr;
                    auto word = [&](int i) { return i >= 0 && i < int(P.tree_words) ? __ldg(tw + i) : 0u; };
#pragma unroll
                    for (int q = 0; q < NW; ++q) {
                        const int q4 = int(half) * NW + q, nd = q4 * 32 - rec;
                        const uint32_t bits = tw ? __funnelshift_r(word(nd >> 5), word((nd >> 5) + 1), nd & 31) & below(rec + int(rows), q4)
                                                 : below(rec + int(ri) + 1, q4);
                        see[q] = bits | below(rec, q4);
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < NW; ++q) see[q] = 0;
                    for (uint32_t k = 0; k < nb; ++k) {
                        const int at = int(k * box), end = at + int(uint32_t(table[j * nb + k].y) >> 24);
#pragma unroll
                        for (int q = 0; q < NW; ++q) see[q] |= below(end, int(half) * NW + q) & ~below(at, int(half) * NW + q);
                    }
                }
            }
            ok = pf_warp_wait(&done[k_seq(j) % NB], (k_seq(j) / NB) & 1);
            if (!ok) break;
            tc_fence_after();
            float x[NK];
            {
                uint32_t* u = reinterpret_cast<uint32_t*>(x);
#pragma unroll
                for (int q = 0; q < NW; ++q) tc_ld32(lane_addr + slot * 128 + half * 64 + q * 32, u + q * 32);
#pragma unroll
                for (int q = 0; q < NW; ++q) tc_wait_ld(u + q * 32);
            }
            const bool tail = kTail16 && t >= n_first;
            if (tail) {  // the powers of two that the keys were divided by
                const uint32_t jt = t - max(tb, n_first);
                ok = pf_warp_wait(&scaled[jt % kAcScales], (jt / kAcScales) & 1);
                if (!ok) break;
                const uint4* ks = reinterpret_cast<const uint4*>(key_scale + (jt % kAcScales) * 128 + half * NK);
#pragma unroll
                for (int k = 0; k < NK; k += 16) {
                    const uint4 w = ks[k / 16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint32_t u = i < 4 ? w.x : i < 8 ? w.y : i < 12 ? w.z : w.w;
                        x[k + i] *= __uint_as_float(((u >> (i % 4 * 8)) & 255u) << 23);
                    }
                }
            }
            if (part) {
#pragma unroll
                for (int k = 0; k < NK; ++k)
                    if (!((see[k >> 5] >> (k & 31)) & 1)) x[k] = -INFINITY;
            }
            float mx = pf_max64(x);
            if constexpr (HS == 1) mx = fmaxf(mx, pf_max64(x + 64));
            mx *= c2;
            if constexpr (HS == 2) xch[(j & 1) * 256 + half * 128] = mx;
            tc_fence_before();
            pair_sync();  // (P of one half goes over S columns that the other half has read by now)
            if (!ok) break;
            tc_fence_after();
            if constexpr (HS == 2) mx = fmaxf(mx, xch[(j & 1) * 256 + (half ^ 1) * 128]);
            const bool need = mx > m_used + kPfRescale;
            if (j == 0) {
                m_used = fmaxf(mx, -1e30f);
            } else if (__any_sync(0xffffffffu, need)) {
                float alpha = 1.f;
                if (need) {
                    alpha = fast_exp2(m_used - mx);
                    m_used = mx;
                    l *= alpha;
                }
                // O holds the products of the tiles before once the last of them is done.
                ok = pf_warp_wait(&done[v_seq(j - 1) % NB], (v_seq(j - 1) / NB) & 1);
                if (!ok) break;
                tc_fence_after();
#pragma unroll 1
                for (uint32_t cc = 0; cc < D / HS; cc += 32) {
                    uint32_t o[32];
                    tc_ld32(col_o + cc, o);
                    tc_wait_ld(o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                    tc_st32(col_o + cc, o);
                }
                tc_wait_st();
                tc_fence_before();
                pair_sync();  // both halves of O are rescaled before either half of P is handed over
                if (!ok) break;
                tc_fence_after();
            }
            // P = exp2(x c2 - m), its sum, and P over its S (16-bit, two per column). 64 keys at a time go
            // to the tensor core.
            const float mneg = -m_used;
            float s4[4] = {0.f, 0.f, 0.f, 0.f};
            auto exps = [&](int from, int to) {
#pragma unroll
                for (int k = from; k < to; k += 2) {
                    pf_fma2(x[k], x[k + 1], x[k], x[k + 1], c2, mneg);
                    x[k] = fast_exp2(x[k]);
                    x[k + 1] = fast_exp2(x[k + 1]);
                    pf_add2(s4[k & 2], s4[(k & 2) + 1], x[k], x[k + 1]);
                }
            };
            auto store = [&](int from, uint32_t part64) {
                uint32_t pk[32];
                if (tail) {  // P = hi + lo, lo in the other half of the columns that S has left
#pragma unroll
                    for (int i = 0; i < 32; ++i) pk[i] = pf_pack2<true>(x[from + 2 * i], x[from + 2 * i + 1]);
                    tc_st32(lane_addr + slot * 128 + part64 * 32, pk);
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float2 hi = at_unpack<true>(pk[i]);
                        pk[i] = pf_pack2<true>(x[from + 2 * i] - hi.x, x[from + 2 * i + 1] - hi.y);
                    }
                    tc_st32(lane_addr + slot * 128 + 64 + part64 * 32, pk);
                    return;
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) pk[i] = pf_pack2<OB>(x[from + 2 * i], x[from + 2 * i + 1]);
                tc_st32(lane_addr + slot * 128 + part64 * 32, pk);
            };
            auto hand_over = [&](uint64_t* bar) {
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(bar);
            };
            exps(0, 64);
            bool bad = false;
            if (part) {
                ok = pf_warp_wait(&scanned[j % kAcScans], (j / kAcScans) & 1);
                if (!ok) break;
                bad = (bad_flag[(j % kAcScans) * 2 + 1] | (kScanWarps == 2 ? bad_flag[(j % kAcScans) * 2] : 0u)) != 0;
            }
            store(0, half);
            if constexpr (HS == 1) {
                exps(64, 96);
                if (!bad) hand_over(&p_full[slot]);
                exps(96, 128);
                store(64, 1);
                if (!bad) hand_over(&p_half[slot]);
            } else {
                if (!bad) hand_over(half ? &p_half[slot] : &p_full[slot]);
            }
            l += (s4[0] + s4[1]) + (s4[2] + s4[3]);
            if (bad) {
                // Sums of p * v over the infinite and NaN values this row sees, which leave the product.
                float fix[D], pl[NK];
#pragma unroll
                for (int k = 0; k < NK; ++k) pl[k] = x[k];
                uint32_t sl[NW];
#pragma unroll
                for (int q = 0; q < NW; ++q) sl[q] = see[q];
                const uint32_t at = v_seq(j) * U;
                auto nonfinite = [&](uint32_t bits) { return tail ? at_nonfinite<true>(bits) : at_nonfinite<OB>(bits); };
#pragma unroll 1
                for (uint32_t d = 0; d < D; ++d) {
                    float f = 0.f;
#pragma unroll 1
                    for (uint32_t k = 0; k < uint32_t(NK); ++k) {
                        const uint32_t key = half * NK + k, kr = key % VK;
                        const uint16_t bits = *reinterpret_cast<const uint16_t*>(
                            ring + ((at + key / VK) % NU) * kAcUnit + (d / 64) * VK * 128 + kr * 128 +
                            ((((d % 64) / 8) ^ (kr & 7)) << 4) + (d % 8) * 2);
                        if (nonfinite(bits) && ((sl[k >> 5] >> (k & 31)) & 1))
                            f += pl[k] * (tail ? at_unpack<true>(bits).x : at_unpack<OB>(bits).x);
                    }
                    fix[d] = f;
                }
                meet();
                for (uint32_t a = 0; a < U; ++a) {
                    uint16_t* v2 = reinterpret_cast<uint16_t*>(ring + ((at + a) % NU) * kAcUnit);
                    for (uint32_t e = uint32_t(tid - 128); e < kAcUnit / 2; e += 128 * HS)
                        if (nonfinite(v2[e])) v2[e] = 0;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                meet();
                if constexpr (HS == 1) {
                    hand_over(&p_full[slot]);
                    mbar_arrive(&p_half[slot]);
                } else {
                    hand_over(half ? &p_half[slot] : &p_full[slot]);
                }
                ok = ok && pf_warp_wait(&done[v_seq(j) % NB], (v_seq(j) / NB) & 1);
                for (uint32_t turn = 0; turn < uint32_t(HS); ++turn) {  // each part of the keys adds to the whole row
                    tc_fence_after();
                    if (ok && turn == half) {
#pragma unroll 1
                        for (uint32_t cc = 0; cc < D; cc += 32) {
                            uint32_t o[32];
                            tc_ld32(lane_addr + kColO + cc, o);
                            tc_wait_ld(o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) + fix[cc + i]);
                            tc_st32(lane_addr + kColO + cc, o);
                        }
                        tc_wait_st();
                    }
                    tc_fence_before();
                    meet();
                }
                if (!ok) break;
            }
        }
        grid_release();
        if (ok) ok = n == 0 || pf_warp_wait(&done[v_seq(n - 1) % NB], (v_seq(n - 1) / NB) & 1);
        if (HS == 2 && ok) {
            xch[(n & 1) * 256 + half * 128] = l;
            pair_sync();
            l += xch[(n & 1) * 256 + (half ^ 1) * 128];
        }
        if (ok) {
            tc_fence_after();
            const bool valid = r < m_end;
            const uint64_t row_id = (uint64_t(b) * P.width + ri) * P.q_heads + qh;
            const uint64_t id = uint64_t(split) * P.seqs * P.width * P.q_heads + row_id;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            constexpr uint32_t kCol = D / HS;  // columns of this thread
            uint8_t* orow = P.out + uint64_t(b) * P.o_seq + uint64_t(ri) * P.o_row + uint64_t(qh) * P.o_head + half * kCol * 2;
            const bool parts = P.splits > 1;
            uint64_t dst0 = parts ? reinterpret_cast<uint64_t>(P.part_o + id * D + half * kCol) : reinterpret_cast<uint64_t>(orow);
            if (!valid) dst0 = 0;
            // Rows go through shared memory (the ring, which every product has left) so that a warp
            // writes whole lines: 32 lanes with a row each would write 32 lines at a time.
            static_assert(NU * kAcUnit >= 128 * D * 4, "row staging");
            uint8_t* stage = ring + uint32_t(warp - 4) * (32 * kCol * 4);
            auto emit = [&](auto as_parts) {
                constexpr bool kParts = decltype(as_parts)::value;
                constexpr uint32_t kChunks = kCol * (kParts ? 4 : 2) / 16, kSwz = kChunks < 8 ? kChunks - 1 : 7;  // 16-byte chunks
                uint8_t* srow = stage + lane * (kChunks * 16);
#pragma unroll 1
                for (uint32_t cc = 0; cc < kCol; cc += 32) {
                    uint32_t o[32];
                    tc_ld32(col_o + cc, o);
                    tc_wait_ld(o);
#pragma unroll
                    for (uint32_t i = 0; i < (kParts ? 8 : 4); ++i) {
                        uint4 y;
                        if constexpr (kParts) {
                            y = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        } else {  // (a row that sees no key has a zero sum; its product is 0)
                            uint32_t z[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                z[e] = pf_pack2<BF16>(__uint_as_float(o[8 * i + 2 * e]) * inv, __uint_as_float(o[8 * i + 2 * e + 1]) * inv);
                            y = make_uint4(z[0], z[1], z[2], z[3]);
                        }
                        *reinterpret_cast<uint4*>(srow + (((cc / (kParts ? 4 : 8) + i) ^ (lane & kSwz)) << 4)) = y;
                    }
                }
                __syncwarp();
                constexpr uint32_t kPer = kChunks < 32 ? 32 / kChunks : 1, kWide32 = kChunks < 32 ? 1 : kChunks / 32;  // rows at a time; rounds per row
                constexpr uint32_t kBatch = 32 / kPer < 8 ? 32 / kPer : 8;                                             // rounds in flight
                const uint32_t c0 = uint32_t(lane) % kChunks;
#pragma unroll 1
                for (uint32_t r0 = uint32_t(lane) / kChunks; r0 < 32; r0 += kBatch * kPer) {
#pragma unroll
                    for (uint32_t part = 0; part < kWide32; ++part) {
                        uint4 y[kBatch];
                        uint64_t to[kBatch];
                        const uint32_t c = c0 + part * 32;
#pragma unroll
                        for (uint32_t k = 0; k < kBatch; ++k) {
                            const uint32_t rr = r0 + k * kPer;
                            to[k] = __shfl_sync(0xffffffffu, dst0, rr);
                            y[k] = *reinterpret_cast<const uint4*>(stage + rr * (kChunks * 16) + ((c ^ (rr & kSwz)) << 4));
                        }
#pragma unroll
                        for (uint32_t k = 0; k < kBatch; ++k)
                            if (to[k]) reinterpret_cast<uint4*>(to[k])[c] = y[k];
                    }
                }
            };
            if (n && parts) emit(std::true_type{});
            else if (n) emit(std::false_type{});
            else if (valid && !parts)  // nothing to see
                for (uint32_t c = 0; c < kCol / 8; ++c) reinterpret_cast<uint4*>(orow)[c] = make_uint4(0, 0, 0, 0);
            if (valid && half == 0) {
                if (parts) P.part_ml[id] = make_float2(l == 0.f ? -INFINITY : m_used, l);
                else if (P.lse) P.lse[row_id] = l == 0.f ? -INFINITY : (m_used + log2f(l)) * kAtLn2;
            }
        } else {
            if (lane == 0) {
                record_error(P.status, KVM_ERR_TIMEOUT, 135);
                *abort_flag = 1;
            }
            __syncwarp();
            __threadfence_block();
            if constexpr (HS == 2) asm volatile("bar.arrive %0, 64;" ::"r"(pair) : "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
}

}  // namespace kvmb
