// Scratch of the microscaled 4-bit linear on the recording HIP stand-in: from what size rows in
// values are quantised by a launch of their own, and what a call does that gets no memory.
// Run by tests/test_mx4_scratch_host.py.
#include "fake_hip.hpp"
#include "ltx_internal.hpp"

// what fake_hip.hpp leaves out
extern "C" hipError_t hipMemsetAsync(void*, int, size_t, hipStream_t s) {
    return fake::capturing.count(s) ? hipErrorStreamCaptureUnsupported : hipSuccess;
}
extern "C" hipError_t hipMemcpyAsync(void*, const void*, size_t, hipMemcpyKind, hipStream_t st) {
    return fake::capturing.count(st) ? hipErrorStreamCaptureUnsupported : hipSuccess;
}

#define CHECK(cond, ...)                                  \
    do {                                                  \
        if (!(cond)) {                                    \
            std::printf("line %d: %s: ", __LINE__, #cond); \
            std::printf(__VA_ARGS__);                     \
            std::printf("\n");                            \
            std::exit(1);                                 \
        }                                                 \
    } while (0)

static ltx_ctx* context() {
    ltx_ctx* c = nullptr;
    CHECK(ltx_init(0, &c), "%s", ltx_last_error(nullptr));
    return c;
}

static int launches(const char* prefix) {
    int n = 0;
    for (const fake::Op& o : fake::log) n += o.what == "launch" && o.name.rfind(prefix, 0) == 0;
    return n;
}

static const hipStream_t kStream = (hipStream_t)0x77;

static void call(ltx_ctx* c, int M, int K, int N = 4096) {
    char* const x = (char*)(1ull << 36);
    fake::log.clear();
    CHECK(ltx_op_linear_mx4(c, x, nullptr, (uint8_t*)x + (1 << 30), (uint8_t*)x + (2ll << 30), nullptr, x + (3ll << 30), 0, M, N,
                            K, 0, LTX_MODE_F16, kStream),
          "%d x %d: %s", M, K, ltx_last_error(c));
}
// quantised first, and a product of two operands in the form
static bool scratch() {
    return launches("ltx_mx4_quantise_f16") == 1 && launches("ltx_linear_mx4_f16_rows_") == 0 && launches("") == 2;
}
static bool alone() { return launches("ltx_linear_mx4_f16_rows_") == 1 && fake::log.size() == 1; }

// Up to 2^17 values are quantised in the product, more by a launch; up to 16 rows always in it.
static void threshold() {
    ltx_ctx* c = context();
    for (int M : {17, 32, 33, 64}) {
        const int K = (1 << 17) / M / 128 * 128;  // the largest that fits
        call(c, M, K);
        CHECK(alone(), "%d x %d", M, K);
        call(c, M, K + 128);
        CHECK(scratch(), "%d x %d", M, K + 128);
    }
    for (int K : {8192, 8320, 16384, 1 << 20}) {
        call(c, 16, K);
        CHECK(alone(), "16 x %d", K);
    }
}

// Without memory, and in a capture, the call that would take scratch goes without.
static void fallback(int captured) {
    ltx_ctx* c = context();
    for (int M : {17, 40, 64}) {
        ltx_ctx* with = context();
        call(with, M, 16384);
        CHECK(scratch(), "with memory, %d rows", M);
        if (captured)
            fake::capturing.insert(kStream);
        else
            fake::limit = fake::in_use;
        call(c, M, 16384);
        CHECK(alone() && !fake::broken_capture, "%d rows: %zu, %s", M, fake::log.size(), fake::log.back().name.c_str());
        fake::capturing.clear();
        fake::limit = ~0ull;
    }
    // and takes it again as soon as there is some
    call(c, 40, 16384);
    CHECK(scratch(), "afterwards");
}

int main(int argc, char** argv) {
    const std::string cmd = argc > 1 ? argv[1] : "";
    if (cmd == "threshold")
        threshold();
    else if (cmd == "no_memory")
        fallback(0);
    else if (cmd == "captured")
        fallback(1);
    else
        CHECK(false, "unknown command %s", cmd.c_str());
    std::printf("ok\n");
    std::fflush(stdout);
    std::_Exit(0);  // (the library's own teardown belongs to the real runtime)
}
