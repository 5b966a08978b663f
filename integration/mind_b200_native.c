/*
 * mind_b200_native.c -- link-time definitions of MIND's deterministic BLAS intrinsics that
 * forward to libmind_b200.so (NVIDIA B200).
 *
 * How it is used.  A MIND project lists this file under `[targets.<name>].native_sources`
 * (src/project/mod.rs:525-540 of star-ga/mind): mindc compiles it with its own deterministic
 * clang invocation and links the object into the executable (src/project/mod.rs:1104-1135),
 * next to `-ldl -lpthread -lm`, which its Linux link line already carries
 * (src/project/link.rs:113-115).  Every `func.call @__mind_blas_*` that the lowering leaves as
 * an external call is then resolved by the definitions below.  They load libmind_b200.so on
 * first use -- from the path in the environment variable MIND_B200_LIB, else by the name
 * "libmind_b200.so" through the normal library search -- and forward the call unchanged: same
 * names, same i64 arguments, same meaning (include/mind_b200.h of the mind-b200 tree names the
 * reference file and line each one replaces).
 *
 * Nothing here computes.  If the library cannot be loaded, or has no usable GPU, the kernels
 * return a negative status (the library's MIND_B200_ERR_* codes; -3 = no device / no library)
 * and the dots return 0, as the reference's dot does on bad input
 * (runtime-support/mind_intrinsics.c:1538); mind_b200_native_last_error() gives the reason.
 * There is no CPU fallback on purpose: a caller that wants the CPU kernels simply does not
 * list this file.
 *
 * A library older than the products of quantised language models serves everything else; those
 * return -3 with it.
 *
 * C99 + POSIX (dlopen, pthread_once) + __thread; no CUDA headers are needed to compile it.
 */
#include <dlfcn.h>
#include <pthread.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#define MIND_B200_NATIVE_NO_LIBRARY (-3)

typedef int64_t (*fn13_t)(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                          int64_t, int64_t, int64_t);
typedef int64_t (*fn12_t)(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                          int64_t, int64_t);
typedef int64_t (*fn9_t)(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t);
typedef int64_t (*fn7_t)(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t);
typedef int64_t (*fn6_t)(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t);
typedef int64_t (*fn5_t)(int64_t, int64_t, int64_t, int64_t, int64_t);
typedef int64_t (*fn3_t)(int64_t, int64_t, int64_t);
typedef const char *(*err_t)(void);

static struct {
    void *handle;
    fn6_t mm_i8, mm_i8_mt, mm_q16, mm_q16_mt, mm_i16;
    fn5_t gemv_q16_mt, rmajor_q16, rmajor_i16;
    fn3_t dot_q16, dot_l1_q16, dot_i16;
    fn13_t w4_grouped_i8, w4_grouped_i16, w4_grouped_q16;
    fn12_t mm_grouped_i8, mm_grouped_i8_bt;
    fn9_t w4_i8, w4_i16, w4_q16;
    fn7_t expert_plan;
    err_t last_error;
    char load_error[512];
} g_b200;

static pthread_once_t g_b200_once = PTHREAD_ONCE_INIT;

static void *b200_sym(const char *name) {
    void *p = dlsym(g_b200.handle, name);
    if (!p && !g_b200.load_error[0])
        snprintf(g_b200.load_error, sizeof g_b200.load_error, "libmind_b200: missing symbol %s", name);
    return p;
}

/* A name that older libraries lack: only calls of it are refused then. */
static void *b200_newer_sym(const char *name) { return dlsym(g_b200.handle, name); }

static void b200_load(void) {
    const char *path = getenv("MIND_B200_LIB");
    if (!path || !*path) path = "libmind_b200.so";
    g_b200.handle = dlopen(path, RTLD_NOW | RTLD_LOCAL);
    if (!g_b200.handle) {
        const char *why = dlerror();
        snprintf(g_b200.load_error, sizeof g_b200.load_error, "cannot load %s: %s", path, why ? why : "unknown error");
        return;
    }
    g_b200.mm_i8 = (fn6_t)b200_sym("__mind_blas_matmul_mm_i8_v");
    g_b200.mm_i8_mt = (fn6_t)b200_sym("__mind_blas_matmul_mm_i8_mt_v");
    g_b200.mm_q16 = (fn6_t)b200_sym("__mind_blas_matmul_mm_q16_v");
    g_b200.mm_q16_mt = (fn6_t)b200_sym("__mind_blas_matmul_mm_q16_mt_v");
    g_b200.mm_i16 = (fn6_t)b200_sym("__mind_b200_matmul_mm_i16");
    g_b200.gemv_q16_mt = (fn5_t)b200_sym("__mind_blas_gemv_q16_mt");
    g_b200.rmajor_q16 = (fn5_t)b200_sym("__mind_blas_matmul_rmajor_q16_v");
    g_b200.rmajor_i16 = (fn5_t)b200_sym("__mind_blas_matmul_rmajor_i16_v");
    g_b200.dot_q16 = (fn3_t)b200_sym("__mind_blas_dot_q16_v");
    g_b200.dot_l1_q16 = (fn3_t)b200_sym("__mind_blas_dot_l1_q16_v");
    g_b200.dot_i16 = (fn3_t)b200_sym("__mind_blas_dot_i16_v");
    g_b200.w4_i8 = (fn9_t)b200_newer_sym("__mind_b200_gemv_w4_i8");
    g_b200.w4_i16 = (fn9_t)b200_newer_sym("__mind_b200_gemv_w4_i16");
    g_b200.w4_q16 = (fn9_t)b200_newer_sym("__mind_b200_gemv_w4_q16");
    g_b200.w4_grouped_i8 = (fn13_t)b200_newer_sym("__mind_b200_gemv_w4_grouped_i8");
    g_b200.w4_grouped_i16 = (fn13_t)b200_newer_sym("__mind_b200_gemv_w4_grouped_i16");
    g_b200.w4_grouped_q16 = (fn13_t)b200_newer_sym("__mind_b200_gemv_w4_grouped_q16");
    g_b200.mm_grouped_i8 = (fn12_t)b200_newer_sym("__mind_b200_matmul_grouped_i8");
    g_b200.mm_grouped_i8_bt = (fn12_t)b200_newer_sym("__mind_b200_matmul_grouped_i8_bt");
    g_b200.expert_plan = (fn7_t)b200_newer_sym("__mind_b200_expert_plan");
    g_b200.last_error = (err_t)b200_sym("mind_b200_last_error");
}

static __thread const char *t_b200_lacks; /* what this thread's last call was refused for, or NULL */

static int b200_ready(void) {
    pthread_once(&g_b200_once, b200_load);
    t_b200_lacks = NULL;
    return g_b200.handle && !g_b200.load_error[0];
}

static int b200_lacks(const char *why) {
    t_b200_lacks = why;
    return 0;
}
#define B200_HAS(name, slot) \
    (b200_ready() && (g_b200.slot || b200_lacks("libmind_b200: this library is older than " #name)))

/* Why the last call of this thread's library failed, or why the library could not be loaded;
 * NULL when there is nothing to report. */
const char *mind_b200_native_last_error(void) {
    pthread_once(&g_b200_once, b200_load);
    if (g_b200.load_error[0]) return g_b200.load_error;
    if (t_b200_lacks) return t_b200_lacks;
    return g_b200.last_error ? g_b200.last_error() : NULL;
}

#define FORWARD6(name, slot)                                                                        \
    int64_t name(int64_t a, int64_t b, int64_t c, int64_t m, int64_t k, int64_t n) {                \
        return b200_ready() ? g_b200.slot(a, b, c, m, k, n) : MIND_B200_NATIVE_NO_LIBRARY;          \
    }
#define FORWARD5(name, slot)                                                                        \
    int64_t name(int64_t w, int64_t x, int64_t y, int64_t rows, int64_t cols) {                     \
        return b200_ready() ? g_b200.slot(w, x, y, rows, cols) : MIND_B200_NATIVE_NO_LIBRARY;       \
    }
#define FORWARD3(name, slot)                                                                        \
    int64_t name(int64_t a, int64_t b, int64_t len) { return b200_ready() ? g_b200.slot(a, b, len) : 0; }

/* int8 GEMM: src/mlir/lowering.rs:7687-7752 and its _mt twin :10368 */
FORWARD6(__mind_blas_matmul_mm_i8_v, mm_i8)
FORWARD6(__mind_blas_matmul_mm_i8_mt_v, mm_i8_mt)
/* Q16.16 GEMM: src/mlir/lowering.rs:9300-9407 and :10019-10341 */
FORWARD6(__mind_blas_matmul_mm_q16_v, mm_q16)
FORWARD6(__mind_blas_matmul_mm_q16_mt_v, mm_q16_mt)
/* int16 GEMM: no counterpart in the reference (new name) */
FORWARD6(__mind_b200_matmul_mm_i16, mm_i16)
/* Q16.16 GEMV and row-major matrix x vector: src/mlir/lowering.rs:10019-10032, :6675, :10723 */
FORWARD5(__mind_blas_gemv_q16_mt, gemv_q16_mt)
FORWARD5(__mind_blas_matmul_rmajor_q16_v, rmajor_q16)
FORWARD5(__mind_blas_matmul_rmajor_i16_v, rmajor_i16)
/* dots: src/mlir/lowering.rs:5695-5830, :6057, :5861-6033 */
FORWARD3(__mind_blas_dot_q16_v, dot_q16)
FORWARD3(__mind_blas_dot_l1_q16_v, dot_l1_q16)
FORWARD3(__mind_blas_dot_i16_v, dot_i16)

/* products of quantised language models: no counterpart in the reference (new names) */
#define FORWARD13(name, slot)                                                                                        \
    int64_t name(int64_t w, int64_t s, int64_t x, int64_t r, int64_t o, int64_t y, int64_t m, int64_t rows,          \
                 int64_t cols, int64_t group, int64_t shift, int64_t experts, int64_t x_rows) {                      \
        return B200_HAS(name, slot) ? g_b200.slot(w, s, x, r, o, y, m, rows, cols, group, shift, experts, x_rows)    \
                                    : MIND_B200_NATIVE_NO_LIBRARY;                                                   \
    }
#define FORWARD12(name, slot)                                                                                        \
    int64_t name(int64_t a, int64_t r, int64_t b, int64_t o, int64_t s, int64_t c, int64_t m, int64_t k, int64_t n,  \
                 int64_t experts, int64_t a_rows, int64_t shift) {                                                   \
        return B200_HAS(name, slot) ? g_b200.slot(a, r, b, o, s, c, m, k, n, experts, a_rows, shift)                 \
                                    : MIND_B200_NATIVE_NO_LIBRARY;                                                   \
    }
#define FORWARD9(name, slot)                                                                                         \
    int64_t name(int64_t w, int64_t s, int64_t x, int64_t y, int64_t tokens, int64_t rows, int64_t cols,             \
                 int64_t group, int64_t shift) {                                                                     \
        return B200_HAS(name, slot) ? g_b200.slot(w, s, x, y, tokens, rows, cols, group, shift)                      \
                                    : MIND_B200_NATIVE_NO_LIBRARY;                                                   \
    }
FORWARD9(__mind_b200_gemv_w4_i8, w4_i8)
FORWARD9(__mind_b200_gemv_w4_i16, w4_i16)
FORWARD9(__mind_b200_gemv_w4_q16, w4_q16)
FORWARD13(__mind_b200_gemv_w4_grouped_i8, w4_grouped_i8)
FORWARD13(__mind_b200_gemv_w4_grouped_i16, w4_grouped_i16)
FORWARD13(__mind_b200_gemv_w4_grouped_q16, w4_grouped_q16)
FORWARD12(__mind_b200_matmul_grouped_i8, mm_grouped_i8)
FORWARD12(__mind_b200_matmul_grouped_i8_bt, mm_grouped_i8_bt)
int64_t __mind_b200_expert_plan(int64_t ids, int64_t offsets, int64_t rows, int64_t place, int64_t count, int64_t experts,
                                int64_t per) {
    return B200_HAS(__mind_b200_expert_plan, expert_plan)
               ? g_b200.expert_plan(ids, offsets, rows, place, count, experts, per)
               : MIND_B200_NATIVE_NO_LIBRARY;
}
