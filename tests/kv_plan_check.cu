// Host-side check of what the attention kernels work out from a batch's lengths
// (no GPU needed).  Built and run by tests/test_kv_plans.py.
#include "../tier_b200/csrc/tk_kvattn_tc.cu"

#include <cstdio>

// the library's other translation units, reduced to what the kernels link against
namespace tk {
tk_status fail(tk_status st, const std::string&) { return st; }
tk_status cuda_fail(cudaError_t e, const char*) { return e == cudaSuccess ? TK_OK : TK_ERR_CUDA; }
int prof_begin(tk_ctx*, cudaStream_t) { return -1; }
void prof_end(tk_ctx*, cudaStream_t, int, int) {}
tk_status ws_ensure(tk_ctx*, size_t, cudaStream_t) { return TK_OK; }
}  // namespace tk

using namespace tk;

static int g_bad = 0;
#define CHECK(cond, ...)                        \
    do {                                        \
        if (!(cond)) {                          \
            ++g_bad;                            \
            if (g_bad < 20) {                   \
                printf("FAIL %s: ", #cond);     \
                printf(__VA_ARGS__);            \
                printf("\n");                   \
            }                                   \
        }                                       \
    } while (0)

// the first key that a row at `pos` sees lies at max(pos - window + 1, 0): in 64 bits
static void first_keys() {
    const int far = 1 << 30, most = 2147483647;
    const int windows[] = {0, 1, 2, 63, 64, 1000, far - 1, far, far + 1, most - 8, most - 1, most};
    const int places[] = {-most, -far, -1000, -6, -4, -1, 0, 1, 62, 63, 64, 999, 1000, far - 2, far - 1};
    for (int w : windows)
        for (int p : places) {
            const long at = p < 0 ? 0 : p;                         // rows before the cache see nothing; the next is at 0
            const long want = w > 0 && at - w + 1 > 0 ? at - w + 1 : 0;
            CHECK(kv_first_key(p, w) == want, "position %d window %d: %d, not %ld", p, w, kv_first_key(p, w), want);
        }
}

// parts are only taken where all of them have a place in the workspace (one an SM), whatever the contents of q_start
static void divisions() {
    for (long sets : {0L, 1L, 2L, 9L, 10L, 74L, 75L, 1L << 20, 1L << 27, 1L << 28, (1L << 28) + 1, 1L << 29, 1L << 31, 1L << 40})
        for (int heads : {1, 2, 8, 65535})
            CHECK(kt::cuts(sets, heads, 148) == ((double)sets * heads <= 74.0), "%ld sets, %d heads", sets, heads);
}

int main() {
    first_keys();
    divisions();
    printf("%d failures\n", g_bad);
    return g_bad != 0;
}
