// Host-side check of what the attention kernels work out from a batch's lengths
// (no GPU needed).  Built and run by tests/test_kv_plans.py.
#include "../tier_b200/csrc/tk_kv.cuh"

#include <cstdio>

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

int main() {
    first_keys();
    printf("%d failures\n", g_bad);
    return g_bad != 0;
}
