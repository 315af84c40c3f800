// Decodes and fused steps whose host memory runs out: an error, no exception across the
// C ABI.  Allocations of chosen sizes fail, on this thread and while armed only: sizes
// of what the library keeps per row, which the HIP runtime does not ask for.  One
// PASS/FAIL line per check.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <new>
#include <vector>

#include "sa_amd.h"

namespace {
thread_local size_t fail_size = 0;
thread_local int failed = 0;
}  // namespace

void* operator new(size_t n) {
    if (fail_size && n == fail_size) {
        ++failed;
        throw std::bad_alloc();
    }
    if (void* p = std::malloc(n ? n : 1)) return p;
    throw std::bad_alloc();
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, size_t) noexcept { std::free(p); }

namespace {

int bad = 0;
void check(bool ok, const char* what, const char* which, size_t size) {
    std::printf("%s %s, %s cache, %zu bytes\n", ok ? "PASS" : "FAIL", what, which, size);
    std::fflush(stdout);
    bad += !ok;
}

template <class T>
T* device(size_t n) {
    void* p = nullptr;
    if (hipMalloc(&p, n * sizeof(T)) != hipSuccess || hipMemset(p, 0, n * sizeof(T)) != hipSuccess) std::exit(2);
    return static_cast<T*>(p);
}

}  // namespace

int main() {
    constexpr int N = 1237, D = 64;   // rows; of one KV head and one page each
    const size_t sizes[] = {N, 4 * N, 16 * N};   // a byte, an integer and a range per row
    for (sa_dtype kv : {SA_DTYPE_F32, SA_DTYPE_BF16, SA_DTYPE_FP8}) {
        const char* name = kv == SA_DTYPE_F32 ? "fp32" : kv == SA_DTYPE_BF16 ? "bf16" : "8-bit";
        const sa_kv_desc desc = {1, 1, D, N, 1, N, kv};
        sa_kvcache* cache = nullptr;
        if (sa_kvcache_create(&desc, &cache) != SA_OK) return 2;
        std::vector<int32_t> rows(N);
        for (int r = 0; r < N; ++r) {
            rows[r] = r;
            if (sa_kvcache_reserve(cache, r, 64, nullptr) != SA_OK || sa_kvcache_set_len(cache, r, 5, nullptr) != SA_OK)
                return 2;
        }
        const size_t ws_bytes = sa_paged_decode_ws_bytes(cache, N, 1) + 16;
        float* q = device<float>((size_t)N * D);
        float* out = device<float>((size_t)N * D);
        char* ws = device<char>(ws_bytes);
        auto decode = [&] {
            return sa_paged_decode(cache, 0, q, N, rows.data(), 1, 0, 1.f, out, ws, ws_bytes, nullptr);
        };
        auto step = [&] {
            return sa_append_decode(cache, 0, q, q, q, N, rows.data(), 1, nullptr, nullptr, 1e-6f, nullptr, nullptr, 0, 1.f,
                                    out, nullptr, ws, ws_bytes, 0, nullptr);
        };
        auto partials = [&] {
            return sa_append_decode_partials(cache, 0, device<float>((size_t)N * 3 * D), 1, N, rows.data(), 1, nullptr,
                                             nullptr, 1e-6f, nullptr, nullptr, 0, 1.f, out, nullptr, ws, ws_bytes, 0,
                                             nullptr);
        };
        auto run = [&](const char* what, auto&& call) {
            int seen = 0;
            for (size_t size : sizes) {
                fail_size = size;
                failed = 0;
                const sa_status st = call();
                fail_size = 0;
                seen += failed;
                check(st == (failed ? SA_ENOMEM : SA_OK), what, name, size);
            }
            check(seen > 0 && call() == SA_OK && hipDeviceSynchronize() == hipSuccess, what, name, 0);
        };
        run("decode", decode);
        run("step", step);
        run("step from partials", partials);
        check(sa_kvcache_len(cache, N - 1) == 5, "lengths", name, 0);
        if (sa_kvcache_destroy(cache) != SA_OK) return 2;
    }
    return bad ? 1 : 0;
}
