// Launcher of the tcgen05 decode-attention kernels (attend_tc.cuh), instantiated
// per type in attend_tc_<type>.cu.
#pragma once
#include "attend_tc.cuh"
#include "lse_launch.cuh"

namespace kvmb {

template <int D, bool BF16, int MODE>
int launch_attend_tc_k(kvm_ctx* c, const AttendTcMaps& maps, const AttendParams& p, uint32_t box, cudaStream_t s) {
    auto fn = attend_tc_kernel<D, BF16, MODE>;
    if constexpr (!ac_wide(D)) {
        // The register split needs every register of 256 x 128: with fewer the warps would wait for more for ever.
        static const int regs = [&] {
            cudaFuncAttributes a{};
            return cudaFuncGetAttributes(&a, fn) == cudaSuccess ? a.numRegs : 0;
        }();
        if (regs != 128) return KVM_ERR_CUDA;
    }
    constexpr uint32_t smem = ac_smem_bytes(D, MODE);
    if (smem_attr(reinterpret_cast<const void*>(fn), int(smem)) != cudaSuccess) return KVM_ERR_CUDA;
    const uint64_t grid = uint64_t(p.seqs) * p.kv_heads * p.m_tiles * p.splits;
    if (grid > 0x7fffffffull) return KVM_ERR_LENGTH;
    fn<<<uint32_t(grid), ac_threads(D), smem, s>>>(maps, p, box);
    ++c->launches;
    return cudaGetLastError() == cudaSuccess ? KVM_OK : KVM_ERR_CUDA;
}

template <bool BF16>
int launch_attend_tc_t(kvm_ctx* c, const AttendTcMaps& maps, const AttendParams& p, uint32_t dim, int mode, uint32_t box,
                       cudaStream_t s) {
    const bool w = mode == kAtWindow;
    switch (dim) {
        case 64: return w ? launch_attend_tc_k<64, BF16, kAtWindow>(c, maps, p, box, s) : launch_attend_tc_k<64, BF16, kAtTree>(c, maps, p, box, s);
        case 128: return w ? launch_attend_tc_k<128, BF16, kAtWindow>(c, maps, p, box, s) : launch_attend_tc_k<128, BF16, kAtTree>(c, maps, p, box, s);
        default: return w ? launch_attend_tc_k<256, BF16, kAtWindow>(c, maps, p, box, s) : launch_attend_tc_k<256, BF16, kAtTree>(c, maps, p, box, s);
    }
}

extern template int launch_attend_tc_t<false>(kvm_ctx*, const AttendTcMaps&, const AttendParams&, uint32_t, int, uint32_t,
                                              cudaStream_t);
extern template int launch_attend_tc_t<true>(kvm_ctx*, const AttendTcMaps&, const AttendParams&, uint32_t, int, uint32_t,
                                             cudaStream_t);

}  // namespace kvmb
