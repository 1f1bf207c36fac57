// Launches that the CUDA runtime refuses, by a fake of its calls (linked with
// --wrap): no device is needed and none is used.  A call that has returned the
// error leaves none behind for the next call to find, and a call that launches
// does not return what somebody else left.
#include <cstdio>
#include "tk_internal.h"

static cudaError_t next = cudaSuccess, left = cudaSuccess;
extern "C" cudaError_t __wrap_cudaLaunchKernelExC(const cudaLaunchConfig_t*, const void*, void**) {
    if (next != cudaSuccess) left = next;
    return next;
}
extern "C" cudaError_t __wrap_cudaGetLastError() {
    const cudaError_t e = left;
    left = cudaSuccess;
    return e;
}
extern "C" cudaError_t __wrap_cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }

int main() {
    tk_ctx c;
    c.num_sms = 148;
    alignas(32) static float x[64], y[64], v[4];
    alignas(32) static int32_t ids[64];
    const struct { const char* name; tk_status (*call)(tk_ctx*, float*, float*, float*, int32_t*); } calls[] = {
        {"tk_logprobs", [](tk_ctx* c, float* x, float*, float* v, int32_t* ids) {
            return tk_logprobs(c, 1, 64, x, 0, 64, ids, 1.0f, v, nullptr, nullptr, nullptr, 0, nullptr, nullptr, nullptr); }},
        {"tk_logprobs, top_k", [](tk_ctx* c, float* x, float*, float* v, int32_t* ids) {
            return tk_logprobs(c, 1, 64, x, 0, 64, ids, 1.0f, v, nullptr, nullptr, nullptr, 4, ids, nullptr, nullptr); }},
        {"tk_logprobs_grad", [](tk_ctx* c, float* x, float* y, float* v, int32_t* ids) {
            return tk_logprobs_grad(c, 1, 64, x, 0, 64, ids, 1.0f, v, v, v, nullptr, nullptr, y, 0, 64, nullptr); }},
        {"tk_distill", [](tk_ctx* c, float* x, float* y, float* v, int32_t* ids) {
            return tk_distill(c, 1, 64, x, 0, 64, 4, ids, x, 1.0f, nullptr, v, nullptr, nullptr, y, 0, 64, nullptr); }},
        {"tk_distill, the loss alone", [](tk_ctx* c, float* x, float*, float* v, int32_t* ids) {
            return tk_distill(c, 1, 64, x, 0, 64, 4, ids, x, 1.0f, nullptr, v, nullptr, nullptr, nullptr, 0, 0, nullptr); }},
        {"tk_distill_grad", [](tk_ctx* c, float* x, float* y, float* v, int32_t* ids) {
            return tk_distill_grad(c, 1, 64, x, 0, 64, 4, ids, x, 1.0f, v, v, nullptr, y, 0, 64, nullptr); }},
    };
    int failures = 0;
    for (const auto& a : calls) {
        for (const auto& b : calls) {                   // refused, then launched
            next = cudaErrorLaunchOutOfResources;
            left = cudaSuccess;
            const tk_status one = a.call(&c, x, y, v, ids);
            next = cudaSuccess;
            const cudaError_t behind = left;
            const tk_status two = b.call(&c, x, y, v, ids);
            if (one == TK_ERR_CUDA && behind == cudaSuccess && two == TK_OK) continue;
            ++failures;
            printf("%s refused: status %d, %s left behind; then %s: status %d\n", a.name, (int)one, cudaGetErrorName(behind), b.name, (int)two);
        }
        left = cudaErrorInvalidValue;                   // not this call's
        const tk_status st = a.call(&c, x, y, v, ids);
        if (st == TK_OK) continue;
        ++failures;
        printf("%s after another's error: status %d\n", a.name, (int)st);
    }
    printf("%d failures\n", failures);
    return failures != 0;
}
