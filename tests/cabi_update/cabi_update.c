/* SPDX-License-Identifier: Apache-2.0
 *
 * TEST PROGRAM: drives the kernels that change weights from plain C through include/fstx_update.h only
 * -- no Python, no torch, no C++ types.  Device memory comes from the HIP runtime's C API.
 *
 * Merges a rank-2 update into an fp32 weight (in place, on a stream), once more with a rank that needs a workspace,
 * and orthogonalises a small and a larger matrix with a step whose result is known; checks everything against loops on
 * the host, and the refusals.  Prints "cabi_update: ok".
 */
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>

#include "fstx_update.h"

typedef int hipError_t;
typedef void *hipStream_t;
enum { hipSuccess = 0, hipMemcpyHostToDevice = 1, hipMemcpyDeviceToHost = 2 };
hipError_t hipSetDevice(int device);
hipError_t hipMalloc(void **ptr, size_t size);
hipError_t hipFree(void *ptr);
hipError_t hipMemcpy(void *dst, const void *src, size_t size, int kind);
hipError_t hipStreamCreate(hipStream_t *stream);
hipError_t hipStreamSynchronize(hipStream_t stream);
hipError_t hipStreamDestroy(hipStream_t stream);

#define CHECK(cond)                                                              \
    do {                                                                         \
        if (!(cond)) {                                                           \
            fprintf(stderr, "cabi_update: FAILED at line %d: %s\n", __LINE__, #cond); \
            return 1;                                                            \
        }                                                                        \
    } while (0)

static uint32_t state = 12345;
static float next(void) { /* -1 .. 1 */
    state = state * 1664525u + 1013904223u;
    return (float)(int32_t)state / 2147483648.0f;
}

static float *on_device(const float *host, size_t n) {
    void *p = NULL;
    if (hipMalloc(&p, n * sizeof(float)) != hipSuccess) return NULL;
    if (host && hipMemcpy(p, host, n * sizeof(float), hipMemcpyHostToDevice) != hipSuccess) return NULL;
    return p;
}

static int merge(uint64_t m, uint64_t n, uint64_t r, hipStream_t stream) {
    float *w = malloc(m * n * 4), *u = malloc(m * r * 4), *d = malloc(r * n * 4), *got = malloc(m * n * 4);
    CHECK(w && u && d && got);
    for (uint64_t i = 0; i < m * n; ++i) w[i] = next();
    for (uint64_t i = 0; i < m * r; ++i) u[i] = next();
    for (uint64_t i = 0; i < r * n; ++i) d[i] = next();
    float *dw = on_device(w, m * n), *du = on_device(u, m * r), *dd = on_device(d, r * n);
    CHECK(dw && du && dd);
    fstx_low_rank_desc desc = {dw, dw, du, dd, NULL, m, n, r, n, n, r, 1, n, 1, 0.5f, FSTX_F32, FSTX_F32, FSTX_F32, 0, 0};
    int64_t need = fstx_merge_low_rank_workspace(&desc, 1);
    CHECK(need >= 0 && (r <= 32 || need > 0));
    float *space = on_device(NULL, (size_t)need / 4 + 64);
    CHECK(space);
    CHECK(need == 0 || fstx_merge_low_rank(&desc, 1, space, (uint64_t)need - 1, stream) == -FSTX_E_INVAL);
    CHECK(fstx_merge_low_rank(&desc, 1, space, (uint64_t)need, stream) == 0);
    CHECK(hipStreamSynchronize(stream) == hipSuccess);
    CHECK(hipMemcpy(got, dw, m * n * 4, hipMemcpyDeviceToHost) == hipSuccess);
    for (uint64_t i = 0; i < m; ++i)
        for (uint64_t j = 0; j < n; ++j) {
            double sum = 0, size = 0;
            for (uint64_t k = 0; k < r; ++k) {
                sum += (double)u[i * r + k] * d[k * n + j];
                size += fabs((double)u[i * r + k] * d[k * n + j]);
            }
            /* six products per k summed in 32 bits, 2^-24 of each left out, and the weight added */
            const double want = w[i * n + j] + 0.5 * sum, tol = 0.5 * size * (6.0 * (double)r + 4.0) * 0x1p-23 + 0x1p-23 * (fabs(want) + 1.0);
            CHECK(fabs(got[i * n + j] - want) <= tol);
        }
    desc.type = 77;
    CHECK(fstx_merge_low_rank(&desc, 1, space, (uint64_t)need, stream) == -FSTX_E_INVAL);
    CHECK(hipFree(dw) == hipSuccess && hipFree(du) == hipSuccess && hipFree(dd) == hipSuccess && hipFree(space) == hipSuccess);
    free(w);
    free(u);
    free(d);
    free(got);
    return 0;
}

static int polar(uint64_t m, uint64_t n, hipStream_t stream) {
    /* one step (a, b, c) = (1.5, -0.5, 0) on G whose rows are orthogonal and of one length: every singular value of
     * X = G / |G| is 1 / sqrt(m), so that the result is (1.5 - 0.5 / m) X */
    static const float step[3] = {1.5f, -0.5f, 0.0f};
    float *g = calloc(m * n, 4), *got = malloc(m * n * 4);
    CHECK(g && got && m <= n);
    for (uint64_t i = 0; i < m; ++i) g[i * n + (i * 7) % n] = i % 2 ? -3.0f : 3.0f;
    float *dg = on_device(g, m * n), *dst = on_device(NULL, m * n);
    CHECK(dg && dst);
    fstx_orthogonalize_desc desc = {dst, dg, m, n, n, n, 1, FSTX_F32, 0};
    int64_t need = fstx_orthogonalize_workspace(&desc, 1, step, 1);
    CHECK(need > 0);
    float *space = on_device(NULL, (size_t)need / 4);
    CHECK(space);
    CHECK(fstx_orthogonalize(&desc, 1, step, 0, 0.0f, space, (uint64_t)need, stream) == -FSTX_E_INVAL);
    CHECK(fstx_orthogonalize(&desc, 1, step, 1, 0.0f, space, (uint64_t)need, stream) == 0);
    CHECK(hipStreamSynchronize(stream) == hipSuccess);
    CHECK(hipMemcpy(got, dst, m * n * 4, hipMemcpyDeviceToHost) == hipSuccess);
    const double factor = (1.5 - 0.5 / (double)m) / (3.0 * sqrt((double)m));
    for (uint64_t i = 0; i < m * n; ++i) /* one entry per row and column: products of zeros and a few roundings to 22 bits */
        CHECK(fabs(got[i] - factor * g[i]) <= 8 * 0x1p-22 * fabs(factor * g[i]));
    CHECK(hipFree(dg) == hipSuccess && hipFree(dst) == hipSuccess && hipFree(space) == hipSuccess);
    free(g);
    free(got);
    return 0;
}

int main(void) {
    hipStream_t stream = NULL;
    CHECK(hipSetDevice(0) == hipSuccess && hipStreamCreate(&stream) == hipSuccess);
    if (merge(70, 45, 2, stream) || merge(130, 201, 70, stream) || polar(5, 40, stream) || polar(96, 200, stream)) return 1;
    CHECK(hipStreamDestroy(stream) == hipSuccess);
    printf("cabi_update: ok\n");
    return 0;
}
