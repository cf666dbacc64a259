// Entry points of the 8-bit checkpoints (include/custos_hip.h).  The kernels are generated from expressions like
// every other: checkpoint8_source in kernel_gen.cpp.
#include "runtime.hpp"

namespace custos_hip {

namespace {

constexpr uint64_t kStreamBeyond = 64ull << 20;

// The kernel is one of the checkpoint kinds, and the length one a launch can have.
int32_t check_kernel(custos_hip_device* dev, const char* what, const custos_hip_kernel* kernel, Kind kind, size_t n) {
    if (!kernel) return set_error(dev, CUSTOS_HIP_ERR_INVALID_ARGUMENT, std::string(what) + ": null kernel");
    if (kernel->spec.kind != kind)
        return set_error(dev, CUSTOS_HIP_ERR_KIND_MISMATCH, std::string(what) + ": the kernel was compiled as another kind");
    // (of one launch, which has fewer than 2^32 threads)
    if (n > (1ull << 34)) return set_error(dev, CUSTOS_HIP_ERR_TOO_LARGE, std::string(what) + ": more than 2^34 elements");
    return CUSTOS_HIP_OK;
}

Operand flat(const char* name, uint64_t ptr, uint64_t bytes, bool written, size_t element, bool in_place = false) {
    return {name, ptr, 1, bytes, 0, written, element, in_place};
}

uint64_t scale_bytes(size_t n) { return (n + kCheckpoint8Block - 1) / kCheckpoint8Block * sizeof(float); }

int32_t launch(custos_hip_device* dev, custos_hip_kernel* kernel, const uint64_t (&ptrs)[4], int n_ptrs, size_t n, uint64_t mode,
               const Operand* ops, size_t n_ops) {
    uint64_t moved = 0;
    for (size_t i = 0; i < n_ops; i++) moved += ops[i].row_bytes;
    if (moved > kStreamBeyond) mode |= 2;
    hipFunction_t fn = nullptr;
    int32_t rc = entry_point(dev, kernel, EntrySet::Single, &fn);
    if (rc != CUSTOS_HIP_OK) return rc;
    OpArg args[7];
    size_t n_args = 0;
    for (int i = 0; i < n_ptrs; i++) args[n_args++] = {&ptrs[i], 8};
    const uint64_t count = n;
    args[n_args++] = {&count, 8};
    const std::vector<unsigned char>& values = kernel->spec.consts.bytes;
    if (kernel->spec.consts.n_params > 0) args[n_args++] = {values.data(), values.size()};
    args[n_args++] = {&mode, 8};
    Access acc[4];
    for (size_t i = 0; i < n_ops; i++) acc[i] = ops[i].access();
    const uint64_t tile = static_cast<uint64_t>(kCheckpoint8Threads) * kCheckpoint8Unroll * kernel->spec.vec_elems;
    OpLaunch op{};
    op.name = (kernel->code ? kernel->code : kernel)->spec.name.c_str();
    op.func = reinterpret_cast<void*>(fn);
    op.module_fn = true;
    op.kernel = kernel;
    op.grid = dim3(static_cast<unsigned int>((n + tile - 1) / tile));
    op.block = dim3(kCheckpoint8Threads);
    op.args = args;
    op.n_args = n_args;
    op.acc = acc;
    op.n_acc = n_ops;
    return launch_op(dev, op);
}

}  // namespace

}  // namespace custos_hip

using namespace custos_hip;

extern "C" {

int32_t custos_hip_checkpoint8_save(custos_hip_device* dev, custos_hip_kernel* kernel, uint64_t x, uint64_t out, uint64_t codes,
                                    uint64_t scales, size_t n) {
    const char* what = "checkpoint save";
    int32_t rc = check_kernel(dev, what, kernel, Kind::Save8, n);
    if (rc != CUSTOS_HIP_OK) return rc;
    REQUIRE_DEV(dev);
    if (n == 0) return CUSTOS_HIP_OK;
    const size_t es = dtype_size(kernel->spec.dtype);
    Operand ops[4] = {flat("x", x, n * es, false, es, true), flat("codes", codes, n, true, 1), flat("scales", scales, scale_bytes(n), true, 4)};
    size_t n_ops = 3;
    if (out) ops[n_ops++] = flat("out", out, n * es, true, es, true);
    rc = check_operands(dev, what, ops, n_ops);
    if (rc != CUSTOS_HIP_OK) return rc;
    return launch(dev, kernel, {x, out, codes, scales}, 4, n, out ? 1 : 0, ops, n_ops);
}

int32_t custos_hip_checkpoint8_restore(custos_hip_device* dev, custos_hip_kernel* kernel, uint64_t codes, uint64_t scales, uint64_t out,
                                       size_t n) {
    const char* what = "checkpoint restore";
    int32_t rc = check_kernel(dev, what, kernel, Kind::Restore8, n);
    if (rc != CUSTOS_HIP_OK) return rc;
    REQUIRE_DEV(dev);
    if (n == 0) return CUSTOS_HIP_OK;
    const size_t es = dtype_size(kernel->spec.dtype);
    const Operand ops[3] = {flat("codes", codes, n, false, 1), flat("scales", scales, scale_bytes(n), false, 4),
                            flat("out", out, n * es, true, es)};
    rc = check_operands(dev, what, ops, 3);
    if (rc != CUSTOS_HIP_OK) return rc;
    return launch(dev, kernel, {codes, scales, out, 0}, 3, n, 0, ops, 3);
}

int32_t custos_hip_add_unary_grad8(custos_hip_device* dev, custos_hip_kernel* kernel, uint64_t codes, uint64_t scales, uint64_t lhs_grad,
                                   uint64_t out_grad, size_t n, int32_t flags) {
    const char* what = "unary gradient from a checkpoint";
    int32_t rc = check_kernel(dev, what, kernel, Kind::UnaryGrad8, n);
    if (rc != CUSTOS_HIP_OK) return rc;
    if (flags & ~CUSTOS_HIP_GRAD_OVERWRITE) return set_error(dev, CUSTOS_HIP_ERR_INVALID_ARGUMENT, std::string(what) + ": unknown flag");
    REQUIRE_DEV(dev);
    if (n == 0) return CUSTOS_HIP_OK;
    const bool overwrite = (flags & CUSTOS_HIP_GRAD_OVERWRITE) != 0;
    const size_t es = dtype_size(kernel->spec.dtype);
    const Operand ops[4] = {flat("codes", codes, n, false, 1), flat("scales", scales, scale_bytes(n), false, 4),
                            flat("lhs_grad", lhs_grad, n * es, true, es, overwrite), flat("out_grad", out_grad, n * es, false, es, true)};
    rc = check_operands(dev, what, ops, 4);
    if (rc != CUSTOS_HIP_OK) return rc;
    return launch(dev, kernel, {codes, scales, lhs_grad, out_grad}, 4, n, overwrite ? 0 : 1, ops, 4);
}

}  // extern "C"
