// Prompt ingestion (prefill) linear layers on the 5th-generation tensor cores.
//
// out[m, n] = act(x[m, k] . W[n, k]^T + bias[n] + residual[m, n]), fp16 in and out, fp32
// accumulation in tensor memory; without activation and residual the output may be fp32 (logits).  The kernel is assembled from CUTLASS's sm_100 building
// blocks (TMA loads of both operands into shared memory, tcgen05.mma issued by one thread,
// accumulators in TMEM, epilogue reading them back with tcgen05.ld), with bias, GELU and the
// residual add fused into the epilogue so that no intermediate goes through HBM twice.
//
// One CTA per 128x128 output tile and no thread-block cluster: every operand load is a plain TMA
// copy of this CTA's own tile.  (Pairing two SMs on a 256x128 tile measured 9 % faster at 2048
// rows, but a clustered mainloop is not something this library ships: whether such a mainloop
// shares operand loads across the cluster is decided inside the template library, and the decode
// path of the same shared object runs on several GPUs with peer memory mapped.)
//
// The decode path never comes here: at one token per step the layers are memory-bound vector
// products (decode_kernel.cuh).  This file serves the whole-prompt pass, where every weight is
// reused across all prompt positions and the work is a real GEMM.
#include <cuda_runtime.h>

#include "cutlass/cutlass.h"
#include "cute/tensor.hpp"
#include "cutlass/numeric_types.h"
#include "cutlass/gemm/device/gemm_universal_adapter.h"
#include "cutlass/gemm/kernel/gemm_universal.hpp"
#include "cutlass/gemm/collective/collective_builder.hpp"
#include "cutlass/epilogue/collective/collective_builder.hpp"
#include "cutlass/epilogue/fusion/operations.hpp"
#include "cutlass/epilogue/thread/activation.h"
#include "cutlass/util/packed_stride.hpp"

#include "prefill_gemm.h"

namespace cfb {
namespace {

using namespace cute;

template <template <class> class Act, class Out = cutlass::half_t>
struct LinearGemm {
    using Element = cutlass::half_t;
    using LayoutA = cutlass::layout::RowMajor;     // activations [m, k]
    using LayoutB = cutlass::layout::ColumnMajor;  // weight [n, k] row-major == [k, n] column-major
    using LayoutC = cutlass::layout::RowMajor;     // residual / output [m, n]
    static constexpr int Align = 8;                // 16-byte rows: what TMA needs
    static constexpr int AlignOut = 16 / sizeof(Out);
    using TileShape = Shape<_128, _128, _64>;
    using ClusterShape = Shape<_1, _1, _1>;
    using Fusion = cutlass::epilogue::fusion::LinCombPerColBiasEltAct<Act, Out, float, Element, Element, float>;
    using Epilogue = typename cutlass::epilogue::collective::CollectiveBuilder<
        cutlass::arch::Sm100, cutlass::arch::OpClassTensorOp, TileShape, ClusterShape,
        cutlass::epilogue::collective::EpilogueTileAuto, float, float, Element, LayoutC, Align, Out, LayoutC, AlignOut,
        cutlass::epilogue::collective::EpilogueScheduleAuto, Fusion>::CollectiveOp;
    using Mainloop = typename cutlass::gemm::collective::CollectiveBuilder<
        cutlass::arch::Sm100, cutlass::arch::OpClassTensorOp, Element, LayoutA, Align, Element, LayoutB, Align, float,
        TileShape, ClusterShape,
        cutlass::gemm::collective::StageCountAutoCarveout<static_cast<int>(sizeof(typename Epilogue::SharedStorage))>,
        cutlass::gemm::collective::KernelScheduleAuto>::CollectiveOp;
    using Kernel = cutlass::gemm::kernel::GemmUniversal<Shape<int, int, int, int>, Mainloop, Epilogue>;
    using Gemm = cutlass::gemm::device::GemmUniversalAdapter<Kernel>;

    static const char* run(const void* x, const void* w, const void* bias, const void* residual, void* out, int m,
                           int n, int k, cudaStream_t st) {
        using StrideA = typename Kernel::StrideA;
        using StrideB = typename Kernel::StrideB;
        using StrideC = typename Kernel::StrideC;
        using StrideD = typename Kernel::StrideD;
        const StrideA sa = cutlass::make_cute_packed_stride(StrideA{}, make_shape(m, k, 1));
        const StrideB sb = cutlass::make_cute_packed_stride(StrideB{}, make_shape(n, k, 1));
        const StrideC sc = cutlass::make_cute_packed_stride(StrideC{}, make_shape(m, n, 1));
        const StrideD sd = cutlass::make_cute_packed_stride(StrideD{}, make_shape(m, n, 1));
        typename Gemm::Arguments args{
            cutlass::gemm::GemmUniversalMode::kGemm,
            {m, n, k, 1},
            {static_cast<const Element*>(x), sa, static_cast<const Element*>(w), sb},
            {{}, static_cast<const Element*>(residual), sc, static_cast<Out*>(out), sd}};
        args.epilogue.thread.alpha = 1.0f;
        args.epilogue.thread.beta = residual ? 1.0f : 0.0f;
        args.epilogue.thread.bias_ptr = static_cast<const Element*>(bias);
        Gemm gemm;
        if (gemm.can_implement(args) != cutlass::Status::kSuccess) return "shape or alignment not supported by the GEMM";
        if (Gemm::get_workspace_size(args) != 0) return "unexpected GEMM workspace";
        if (gemm.initialize(args, nullptr, st) != cutlass::Status::kSuccess) return "GEMM initialisation failed";
        if (gemm.run(st) != cutlass::Status::kSuccess) return "GEMM launch failed";
        return nullptr;
    }
};

}  // namespace

const char* prefill_linear(const void* x, const void* w, const void* bias, const void* residual, void* out, int m, int n,
                           int k, int act, cudaStream_t st) {
    switch (act) {
        case PREFILL_ACT_NONE:
            return LinearGemm<cutlass::epilogue::thread::Identity>::run(x, w, bias, residual, out, m, n, k, st);
        case PREFILL_ACT_GELU_TANH:
            return LinearGemm<cutlass::epilogue::thread::GELU_taylor>::run(x, w, bias, residual, out, m, n, k, st);
        case PREFILL_ACT_GELU_ERF:
            return LinearGemm<cutlass::epilogue::thread::GELU>::run(x, w, bias, residual, out, m, n, k, st);
        case PREFILL_OUT_FP32:
            return LinearGemm<cutlass::epilogue::thread::Identity, float>::run(x, w, bias, residual, out, m, n, k, st);
        default:
            return "unknown activation";
    }
}

}  // namespace cfb
