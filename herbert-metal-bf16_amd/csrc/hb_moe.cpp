// hb_moe.cpp -- the routed experts of one MoE layer as one host call: the
// dispatch sequence QwenEngine encodes per prefill block or decode step
// (src/metal/qwen.rs:2705-2735), on the kernels the selection picked
// (hb_engine_experts, expert_pipes qwen.rs:2326-2391).
#include "hb_internal.h"

namespace hb {

// ptr/size: state, route, list, tiles, x, w_gate_up, egu, ehb, w_down, ey,
// xs, out (hb_moe_io's order, then out).
int moe_experts_run(hb_gpu* g, const int32_t kernels[4], int32_t swiglu, int32_t combine,
                    void* const ptr[12], const uint64_t size[12], uint32_t m) {
    enum { STATE, ROUTE, LIST, TILES, X, WGU, EGU, EHB, WDN, EY, XS, OUT };
    const int32_t sort = kernels[0], gu = kernels[1], dn = kernels[2], gather = kernels[3];
    const hb_desc* sd = kernel_desc(g, sort);
    const hb_desc* gd = kernel_desc(g, gu);
    if (!sd || !gd || !kernel_desc(g, dn) || !kernel_desc(g, combine))
        return fail(HB_ERR_INVALID, "moe experts: a kernel of the layer is not built");
    if (sd->kind != HB_KIND_SORT && sd->kind != HB_KIND_SORT_ATOMIC)
        return fail(HB_ERR_INVALID, "moe experts: kernels[0] is not a moe_sort");
    // Grouped expert GEMMs only (never a dense split-K pair, whose
    // workspace the static entry point could not allocate).
    const hb_desc* dd = kernel_desc(g, dn);
    const bool q4 = gd->kind == HB_KIND_MATVEC_Q4, mv_f8 = gd->kind == HB_KIND_MATVEC_F8, f8 = gd->kind == HB_KIND_GEMM_F8;
    if (gd->rows_of == HB_ROWS_DENSE || dd->rows_of == HB_ROWS_DENSE ||
        dd->kind != (q4 || mv_f8 || f8 ? gd->kind : (uint32_t)HB_KIND_GEMM))
        return fail(HB_ERR_INVALID, "moe experts: kernels[1] and kernels[2] are grouped expert GEMMs");
    if ((q4 || mv_f8) && (sd->bm != 16 || gd->rows_of != HB_ROWS_GATHER || dd->rows_of != HB_ROWS_SCATTER || gather >= 0))
        return fail(HB_ERR_INVALID, std::string("moe experts in ") + (q4 ? "4" : "8") +
                                        " bits: a sort of 16-row tiles, gathered gate|up rows, "
                                        "scattered down rows, no gather kernel");
    if (f8) {
        const hb_desc* qd = kernel_desc(g, gather);
        if (sd->bm != gd->bm || sd->bm != dd->bm || gd->rows_of != HB_ROWS_GATHER || dd->rows_of != HB_ROWS_SCATTER ||
            gd->out != HB_OUT_SWIGLU || !qd || qd->kind != HB_KIND_F8_QUANTIZE || qd->form != HB_F8_ROWS || qd->k != gd->k)
            return fail(HB_ERR_INVALID, "moe experts in 8 bits: a sort of the products' tiles, gathered gate|up rows with the "
                                        "SwiGLU, scattered down rows, kernels[3] the quantise kernel of x's rows");
    }
    // The 8-bit products' rows: gate and up's h is down's x, both of the sort's pairs.
    if ((mv_f8 || f8) && (gd->n != 2 * dd->k || gd->k != dd->n || gd->top_k != sd->top_k || dd->top_k != sd->top_k ||
                          gd->experts != sd->experts || dd->experts != sd->experts))
        return fail(HB_ERR_INVALID, "moe experts in 8 bits: kernels of other sizes, experts or top_k than one another's");
    // Its rows would be half as long as the combine reads them.
    if (writes_swiglu(*dd)) return fail(HB_ERR_INVALID, "moe experts: a down kernel that writes a SwiGLU");
    const bool fused = writes_swiglu(*gd);
    if (!fused && !kernel_desc(g, swiglu))
        return fail(HB_ERR_INVALID, "moe experts: the gate|up GEMM needs the swiglu_slots kernel");
    const uint32_t top_k = sd->top_k;
    int rc;
    auto run = [&](int32_t k, std::initializer_list<int> b, uint32_t rows) {
        void* p[8];
        uint64_t s[8];
        uint32_t n = 0;
        for (int i : b) {
            p[n] = ptr[i];
            s[n] = size[i];
            n++;
        }
        return launch_ptrs(g, k, p, s, n, rows);
    };
    if ((rc = run(sort, {STATE, ROUTE, LIST, TILES}, m))) return rc;
    int xin = X;
    if (f8) {
        if ((rc = run(gather, {X, XS}, m))) return rc;
        xin = XS;
    } else if (gather >= 0) {
        if ((rc = run(gather, {STATE, LIST, X, XS}, m))) return rc;
        xin = XS;
    }
    if (fused) {
        // The grouped gate|up writes the SwiGLU of its sums itself.
        if ((rc = run(gu, {STATE, WGU, xin, EHB, LIST, TILES}, m))) return rc;
    } else {
        if ((rc = run(gu, {STATE, WGU, xin, EGU, LIST, TILES}, m))) return rc;
        if ((rc = run(swiglu, {EGU, EHB}, m * top_k))) return rc;
    }
    if ((rc = run(dn, {STATE, WDN, EHB, EY, LIST, TILES}, m))) return rc;
    return run(combine, {EY, ROUTE, OUT}, m);
}

}  // namespace hb

using namespace hb;

extern "C" int hb_moe_experts_run(hb_gpu* g, const int32_t kernels[4], int32_t swiglu,
                                  int32_t combine, const hb_moe_io* io, hb_range out, uint32_t m) {
    const hb_range r[12] = {io->state, io->route, io->list, io->tiles, io->x, io->w_gate_up,
                            io->egu,   io->ehb,   io->w_down, io->ey,  io->xs, out};
    // xs is bound only with a gather, egu only when the SwiGLU is not fused
    // into the gate|up GEMM: otherwise those ranges are not looked at.
    const hb_desc* gd = kernel_desc(g, kernels[1]);
    const bool need_xs = kernels[3] >= 0, need_egu = !gd || !writes_swiglu(*gd);
    void* ptr[12];
    uint64_t size[12];
    for (int i = 0; i < 12; i++) {
        ptr[i] = nullptr;
        size[i] = 0;
        if ((i == 10 && !need_xs) || (i == 6 && !need_egu)) continue;
        char* p = nullptr;
        int rc = resolve(g, r[i], &p, &size[i]);
        if (rc) return rc;
        ptr[i] = p;
    }
    return moe_experts_run(g, kernels, swiglu, combine, ptr, size, m);
}
