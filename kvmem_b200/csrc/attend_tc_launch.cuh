// Launcher of the tcgen05 decode-attention kernels (attend_tc.cuh), instantiated
// per type in attend_tc_<type>.cu.
#pragma once
#include <atomic>

#include "attend_tc.cuh"
#include "lse_launch.cuh"

namespace kvmb {

// KVM_ERR_UNSUPPORTED (nothing launched): this build of the kernel cannot split its registers.
template <int D, bool BF16, int MODE, bool QUANT>
int launch_attend_tc_k(kvm_ctx* c, const AttendTcMaps& maps, const AttendParams& p, uint32_t box, cudaStream_t s) {
    auto fn = attend_tc_kernel<D, BF16, MODE, QUANT>;
    if constexpr (!ac_wide(D) || QUANT) {
        static std::atomic<int> known{0};  // registers of the compiled kernel
        int regs = known.load(std::memory_order_relaxed);
        if (!regs) {
            cudaFuncAttributes a{};
            if (cudaFuncGetAttributes(&a, fn) != cudaSuccess) {
                cudaGetLastError();
                return KVM_ERR_CUDA;
            }
            known.store(regs = a.numRegs, std::memory_order_relaxed);
        }
        if (!ac_registers_fit(QUANT, regs)) return KVM_ERR_UNSUPPORTED;
    }
    constexpr uint32_t smem = ac_smem_bytes(D, MODE, QUANT);
    if (smem_attr(reinterpret_cast<const void*>(fn), int(smem)) != cudaSuccess) return KVM_ERR_CUDA;
    const uint64_t grid = uint64_t(p.seqs) * p.kv_heads * p.m_tiles * p.splits;
    if (grid > 0x7fffffffull) return KVM_ERR_LENGTH;
    fn<<<uint32_t(grid), ac_threads(D, QUANT), smem, s>>>(maps, p, box);
    ++c->launches;
    return cudaGetLastError() == cudaSuccess ? KVM_OK : KVM_ERR_CUDA;
}

template <int D, bool BF16>
int launch_attend_tc_d(kvm_ctx* c, const AttendTcMaps& maps, const AttendParams& p, int mode, bool quant, uint32_t box,
                       cudaStream_t s) {
    if (mode == kAtWindow) return launch_attend_tc_k<D, BF16, kAtWindow, false>(c, maps, p, box, s);
    return quant ? launch_attend_tc_k<D, BF16, kAtTree, true>(c, maps, p, box, s)
                 : launch_attend_tc_k<D, BF16, kAtTree, false>(c, maps, p, box, s);
}

template <bool BF16>
int launch_attend_tc_t(kvm_ctx* c, const AttendTcMaps& maps, const AttendParams& p, uint32_t dim, int mode, bool quant,
                       uint32_t box, cudaStream_t s) {
    switch (dim) {
        case 64: return launch_attend_tc_d<64, BF16>(c, maps, p, mode, quant, box, s);
        case 128: return launch_attend_tc_d<128, BF16>(c, maps, p, mode, quant, box, s);
        default: return launch_attend_tc_d<256, BF16>(c, maps, p, mode, quant, box, s);
    }
}

extern template int launch_attend_tc_t<false>(kvm_ctx*, const AttendTcMaps&, const AttendParams&, uint32_t, int, bool,
                                              uint32_t, cudaStream_t);
extern template int launch_attend_tc_t<true>(kvm_ctx*, const AttendTcMaps&, const AttendParams&, uint32_t, int, bool,
                                             uint32_t, cudaStream_t);

}  // namespace kvmb
