// hb_gemm -- a native host of the C ABI (include/herbert_hip.h): for each
// shape on the command line the selection layer picks a kernel (the
// engine's --tune settings, the [autotune] log on stderr), then the pick is
// timed on this GPU and one line per shape printed.  The inputs come from
// the library's seeded generator (X ~ N(0,1), W ~ N(0,0.02), bf16).
//
//   hb_gemm [--tune key=value,...] [--reps N] SHAPE...
//   SHAPE  MxKxN      a dense GEMM, Y = X.W^T, Out::Bf16
//          MxKxNr     the same with Out::Residual (Y += ...)
//          MxKxNf     the same with Out::F32
//          mv:MxKxN   the decode matvec over M <= 16 rows
//          q4:MxKxN   the same over W quantised to 4 bits, groups of 32
//          f8:MxKxN   W quantised to 8 bits: up to 16 rows the matvec, more the
//                     GEMM, x's rows quantised before it
//
// Output per shape: shape, kernel, microseconds per launch, TFLOP/s (GEMM)
// or GB/s of algorithmic bytes (matvec).  The reference's counterpart is
// its prefill/decode benchmarks driving QwenEngine (src/metal/qwen.rs) with
// --tune; this links the library the same way a Rust host would.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>
#include <vector>

#include "herbert_hip.h"

namespace {

int die(const char* what) {
    fprintf(stderr, "hb_gemm: %s: %s\n", what, hb_last_error());
    return 1;
}

struct Shape {
    bool matvec = false, q4 = false, f8 = false;
    uint32_t m = 0, k = 0, n = 0, out = HB_OUT_BF16;
};

bool parse(const char* s, Shape* sh) {
    if (!strncmp(s, "mv:", 3) || !strncmp(s, "q4:", 3)) {
        sh->matvec = true;
        sh->q4 = *s == 'q';
        s += 3;
    } else if (!strncmp(s, "f8:", 3)) {
        sh->f8 = true;
        s += 3;
    }
    char tail[8] = "";
    if (sscanf(s, "%ux%ux%u%7s", &sh->m, &sh->k, &sh->n, tail) < 3) return false;
    if (!strcmp(tail, "r")) sh->out = HB_OUT_RESIDUAL;
    else if (!strcmp(tail, "f")) sh->out = HB_OUT_F32;
    else if (tail[0]) return false;
    if (sh->f8) sh->matvec = sh->m <= 16;
    return sh->m && sh->k && sh->n && (!sh->matvec || sh->m <= 16);
}

hb_range whole(hb_buf b) {
    hb_range r;
    memset(&r, 0, sizeof r);
    r.buf = b;
    return r;
}

// A buffer of `count` bf16 from the seeded generator.
int normal_buf(hb_gpu* g, uint64_t seed, float std, uint64_t count, hb_buf* out) {
    std::vector<uint16_t> h(count);
    hb_fill_normal_bf16(seed, std, h.data(), count, 8);
    int rc = hb_alloc(g, count * 2, out);
    if (rc) return rc;
    return hb_upload(g, *out, 0, h.data(), count * 2);
}

}  // namespace

int main(int argc, char** argv) {
    std::string tune;
    uint32_t reps = 20;
    std::vector<Shape> shapes;
    for (int i = 1; i < argc; i++) {
        if (!strcmp(argv[i], "--tune") && i + 1 < argc) {
            tune = argv[++i];
        } else if (!strcmp(argv[i], "--reps") && i + 1 < argc) {
            reps = (uint32_t)atoi(argv[++i]);
        } else {
            Shape sh;
            if (!parse(argv[i], &sh)) {
                fprintf(stderr, "hb_gemm: bad shape '%s' (MxKxN[r|f], f8:MxKxN, mv:MxKxN or q4:MxKxN, M <= 16)\n", argv[i]);
                return 2;
            }
            shapes.push_back(sh);
        }
    }
    if (shapes.empty() || !reps) {
        fprintf(stderr, "usage: hb_gemm [--tune key=value,...] [--reps N] MxKxN[r|f] | mv:MxKxN | q4:MxKxN | f8:MxKxN ...\n");
        return 2;
    }
    hb_gpu* g = nullptr;
    if (hb_open(0, &g)) return die("hb_open");
    fprintf(stderr, "[gpu] %s\n", hb_device_summary(g));
    hb_engine* e = nullptr;
    if (hb_engine_open(g, tune.c_str(), &e)) return die("hb_engine_open");
    int status = 0;
    for (const Shape& s : shapes) {
        const uint64_t ysz = (uint64_t)s.m * s.n * (s.out == HB_OUT_F32 ? 4 : 2);
        hb_buf x, w, y, st;
        if (normal_buf(g, 0x5EED0000u + s.k, 1.0f, (uint64_t)s.m * s.k, &x) ||
            normal_buf(g, 0x5EED0001u + s.k, 0.02f, (uint64_t)s.n * s.k, &w) || hb_alloc(g, ysz, &y) ||
            hb_zero(g, y, 0, ysz) || hb_alloc(g, 16, &st))
            return die("buffers");
        const uint32_t state[4] = {0, 0, 0, s.m};
        if (hb_upload(g, st, 0, state, sizeof state)) return die("state");
        int32_t kern = -1;
        hb_op ops[2];
        memset(ops, 0, sizeof ops);
        hb_op& op = ops[0];
        hb_op& second = ops[1];
        uint32_t nops = 1;
        hb_buf rows8 = 0;
        bool have_rows8 = false;
        op.m = second.m = s.m;
        if (s.f8) {
            // W's place is taken by its 8-bit form.
            hb_desc d;
            memset(&d, 0, sizeof d);
            d.kind = HB_KIND_F8_QUANTIZE;
            d.k = s.k;
            d.n = s.n;
            const uint64_t bytes = hb_f8_bytes(s.k, s.n);
            hb_buf q = 0;
            int32_t quant = -1;
            if (hb_kernel_build(g, &d, &quant) || hb_alloc(g, bytes, &q)) {
                status = die("f8");
                continue;
            }
            const hb_range b[2] = {whole(w), whole(q)};
            if (hb_launch(g, quant, b, 2, 1) || hb_sync(g)) return die("f8_quantize");
            hb_free(g, w);
            w = q;
            memset(&d, 0, sizeof d);
            d.kind = s.matvec ? HB_KIND_MATVEC_F8 : HB_KIND_GEMM_F8;
            d.k = s.k;
            d.n = s.n;
            d.out = s.out;
            if (s.matvec) d.mv_m = s.m;
            else d.rows_max = s.m;
            if (hb_kernel_build(g, &d, &kern)) {
                status = die("f8");
                continue;
            }
            if (s.matvec) {
                op.nbind = 3;
                op.bind[0] = whole(w);
                op.bind[1] = whole(x);
                op.bind[2] = whole(y);
            } else {
                hb_desc qd;
                memset(&qd, 0, sizeof qd);
                qd.kind = HB_KIND_F8_QUANTIZE;
                qd.form = HB_F8_ROWS;
                qd.k = s.k;
                if (hb_kernel_build(g, &qd, &op.kernel) || hb_alloc(g, s.m * hb_f8_row_bytes(s.k), &rows8)) {
                    status = die("f8 rows");
                    continue;
                }
                have_rows8 = true;
                op.nbind = 2;
                op.bind[0] = whole(x);
                op.bind[1] = whole(rows8);
                second.nbind = 6;
                const hb_range gb[6] = {whole(st), whole(w), whole(rows8), whole(y), whole(st), whole(st)};
                memcpy(second.bind, gb, sizeof gb);
                second.kernel = kern;
                nops = 2;
            }
        } else if (s.q4) {
            // W's place is taken by its packed form.
            const uint64_t bytes = hb_q4_bytes(s.k, s.n, 32);
            hb_desc d;
            memset(&d, 0, sizeof d);
            d.kind = HB_KIND_Q4_QUANTIZE;
            d.k = s.k;
            d.n = s.n;
            d.bk = 32;
            hb_buf q = 0;
            int32_t quant = -1;
            if (hb_kernel_build(g, &d, &quant) || hb_alloc(g, bytes, &q)) {
                status = die("q4");
                continue;
            }
            const hb_range b[2] = {whole(w), whole(q)};
            if (hb_launch(g, quant, b, 2, 1) || hb_sync(g)) return die("q4_quantize");
            hb_free(g, w);
            w = q;
            const hb_range wr = whole(w);
            if (hb_engine_matvec_q4(e, s.k, s.n, s.out, 32, s.m, &wr, 1, whole(x), whole(y), &kern)) {
                status = die("hb_engine_matvec_q4");
                continue;
            }
            op.nbind = 3;
            op.bind[0] = whole(w);
            op.bind[1] = whole(x);
            op.bind[2] = whole(y);
        } else if (s.matvec) {
            hb_range wr = whole(w);
            if (hb_engine_matvec(e, s.k, s.n, s.out, s.m, &wr, 1, whole(x), whole(y), &kern)) {
                status = die("hb_engine_matvec");
                continue;
            }
            op.nbind = 3;
            op.bind[0] = whole(w);
            op.bind[1] = whole(x);
            op.bind[2] = whole(y);
        } else {
            if (hb_engine_gemm(e, s.k, s.n, s.out, whole(st), whole(w), whole(x), whole(y), s.m, &kern)) {
                status = die("hb_engine_gemm");
                continue;
            }
            op.nbind = 6;
            op.bind[0] = whole(st);
            op.bind[1] = whole(w);
            op.bind[2] = whole(x);
            op.bind[3] = whole(y);
            op.bind[4] = whole(st);
            op.bind[5] = whole(st);
        }
        if (nops == 1) op.kernel = kern;
        double secs = 0;
        if (hb_time(g, ops, nops, 3, &secs) || hb_time(g, ops, nops, reps, &secs)) return die("hb_time");
        const double t = secs / reps;
        if (s.matvec) {
            const double weights = s.q4 ? (double)s.n * s.k * (0.5 + 2.0 / 32) : s.f8 ? (double)hb_f8_bytes(s.k, s.n) : 2.0 * s.n * s.k;
            // Residual reads y too, F32 writes twice the bytes.
            const double bytes = weights + 2.0 * s.m * s.k + 2.0 * s.m * s.n * (s.out == HB_OUT_BF16 ? 1 : 2);
            printf("%s:%ux%ux%u %s %.2f us %.1f GB/s\n", s.q4 ? "q4" : s.f8 ? "f8" : "mv", s.m, s.k, s.n, hb_kernel_name(g, kern), t * 1e6,
                   bytes / t / 1e9);
        } else {
            printf("%s%ux%ux%u%s %s %.2f us %.1f TFLOP/s\n", s.f8 ? "f8:" : "", s.m, s.k, s.n,
                   s.out == HB_OUT_RESIDUAL ? "r" : s.out == HB_OUT_F32 ? "f" : "", hb_kernel_name(g, kern),
                   t * 1e6, 2.0 * s.m * s.n * s.k / t / 1e12);
        }
        fflush(stdout);
        for (hb_buf b : {x, w, y, st}) hb_free(g, b);
        if (have_rows8) hb_free(g, rows8);
    }
    hb_engine_log_summary(e);
    hb_engine_close(e);
    hb_close(g);
    return status;
}
