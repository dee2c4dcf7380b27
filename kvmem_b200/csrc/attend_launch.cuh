// Launcher of the decode-attention kernels (attend.cuh), instantiated once per
// (head_dim, type) in attend_d<dim>_<type>.cu so the variants compile in parallel.
#pragma once
#include "attend.cuh"
#include "lse_launch.cuh"

namespace kvmb {

template <int D, int WM, bool BF16, int MODE, bool QUANT>
int launch_attend_k(kvm_ctx* c, const AttendParams& p, cudaStream_t s) {
    auto fn = attend_mma_kernel<D, WM, BF16, MODE, QUANT>;
    constexpr uint32_t smem = at_smem_bytes(D, WM, QUANT);
    if (smem_attr(reinterpret_cast<const void*>(fn), int(smem)) != cudaSuccess) return KVM_ERR_CUDA;
    const uint64_t grid = uint64_t(p.seqs) * p.kv_heads * p.m_tiles * p.splits;
    if (grid > 0x7fffffffull) return KVM_ERR_LENGTH;
    fn<<<uint32_t(grid), kAtThreads, smem, s>>>(p);
    ++c->launches;
    return cudaGetLastError() == cudaSuccess ? KVM_OK : KVM_ERR_CUDA;
}

template <int D, int WM, bool BF16>
int launch_attend_m(kvm_ctx* c, const AttendParams& p, int mode, bool quant, cudaStream_t s) {
    if (mode == kAtWindow) return launch_attend_k<D, WM, BF16, kAtWindow, false>(c, p, s);
    return quant ? launch_attend_k<D, WM, BF16, kAtTree, true>(c, p, s)
                 : launch_attend_k<D, WM, BF16, kAtTree, false>(c, p, s);
}

template <int D, bool BF16>
int launch_attend_t(kvm_ctx* c, const AttendParams& p, int mode, bool quant, int wm, cudaStream_t s) {
    return wm == 1   ? launch_attend_m<D, 1, BF16>(c, p, mode, quant, s)
           : wm == 2 ? launch_attend_m<D, 2, BF16>(c, p, mode, quant, s)
                     : launch_attend_m<D, 4, BF16>(c, p, mode, quant, s);
}

template <int D, bool BF16>
int launch_attend_combine_t(kvm_ctx* c, const AttendParams& p, cudaStream_t s) {
    const uint64_t rows = uint64_t(p.seqs) * p.width * p.q_heads;
    if (rows > 0x7fffffffull) return KVM_ERR_LENGTH;
    const uint32_t warps = p.splits < 8 ? (p.splits < 4 ? 2 : 4) : 8;
    ++c->launches;
    if (launch_early(attend_combine_kernel<D, BF16>, uint32_t(rows), warps * 32, 0, s, p) == cudaSuccess) return KVM_OK;
    cudaGetLastError();
    return KVM_ERR_CUDA;
}

// The joining pass, where the keys were split.
inline int launch_attend_combine(kvm_ctx* c, const AttendParams& p, uint32_t dim, bool bf16, cudaStream_t s) {
    if (p.splits == 1) return KVM_OK;
    switch (dim) {
        case 64: return bf16 ? launch_attend_combine_t<64, true>(c, p, s) : launch_attend_combine_t<64, false>(c, p, s);
        case 128: return bf16 ? launch_attend_combine_t<128, true>(c, p, s) : launch_attend_combine_t<128, false>(c, p, s);
        default: return bf16 ? launch_attend_combine_t<256, true>(c, p, s) : launch_attend_combine_t<256, false>(c, p, s);
    }
}

extern template int launch_attend_t<64, false>(kvm_ctx*, const AttendParams&, int, bool, int, cudaStream_t);
extern template int launch_attend_t<64, true>(kvm_ctx*, const AttendParams&, int, bool, int, cudaStream_t);
extern template int launch_attend_t<128, false>(kvm_ctx*, const AttendParams&, int, bool, int, cudaStream_t);
extern template int launch_attend_t<128, true>(kvm_ctx*, const AttendParams&, int, bool, int, cudaStream_t);
extern template int launch_attend_t<256, false>(kvm_ctx*, const AttendParams&, int, bool, int, cudaStream_t);
extern template int launch_attend_t<256, true>(kvm_ctx*, const AttendParams&, int, bool, int, cudaStream_t);

}  // namespace kvmb
