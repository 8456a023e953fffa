// Microscaled 4-bit operands, rotary positions and windowed attention on the recording HIP
// stand-in (refusals, scratch, routes), and the window's index arithmetic compiled for the
// host. Run by tests/test_stream_host.py.
#include <algorithm>
#include <cmath>
#include <random>

#include "fake_hip.hpp"
#include "ltx_internal.hpp"
#include "ltx_kv_index.h"

// what fake_hip.hpp leaves out
extern "C" hipError_t hipMemsetAsync(void*, int, size_t, hipStream_t s) {
    return fake::capturing.count(s) ? hipErrorStreamCaptureUnsupported : hipSuccess;
}
static std::vector<char> copied;  // what a host array of a plan became
extern "C" hipError_t hipMemcpyAsync(void*, const void* s, size_t n, hipMemcpyKind kind, hipStream_t st) {
    fake::log.push_back({"copy", "", st});
    if (fake::capturing.count(st)) {
        fake::broken_capture = true;
        return hipErrorStreamCaptureUnsupported;
    }
    if (kind == hipMemcpyHostToDevice) copied.assign((const char*)s, (const char*)s + n);
    return hipSuccess;
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

static char* const X = (char*)(1ull << 36);  // a caller's tensors: aligned addresses
static char* ptr(int i) { return X + ((size_t)i << 30); }

static int launches(const char* prefix) {
    int n = 0;
    for (const fake::Op& o : fake::log) n += o.what == "launch" && o.name.rfind(prefix, 0) == 0;
    return n;
}

#define REFUSED(call, text)                                                                  \
    do {                                                                                     \
        fake::log.clear();                                                                   \
        CHECK(!(call), "taken: %s", #call);                                                  \
        CHECK(std::strstr(ltx_last_error(c), text), "%s: %s", #call, ltx_last_error(c));     \
        CHECK(launches("") == 0, "%s launched", #call);                                      \
    } while (0)

static ltx_ctx* context() {
    ltx_ctx* c = nullptr;
    CHECK(ltx_init(0, &c), "%s", ltx_last_error(nullptr));
    return c;
}

// ---- microscaled operands -----------------------------------------------------------

struct Linear {
    ltx_ctx* c;
    const char *a = ptr(0), *as = ptr(1), *q = ptr(2), *s = ptr(3), *bias = ptr(4);
    char* y = ptr(5);
    int f32 = 0, M = 5, N = 64, K = 256, gelu = 0, mode = LTX_MODE_F16;
    hipStream_t st = nullptr;
    int operator()() const {
        return ltx_op_linear_mx4(c, a, (const uint8_t*)as, (const uint8_t*)q, (const uint8_t*)s, (const float*)bias, y, f32, M,
                                 N, K, gelu, mode, st);
    }
};

static void mx4_refusals() {
    ltx_ctx* c = context();
    auto rows = [&](bool in, char* x, int64_t ld, char* q, char* s, int n, int K, int mode) {
        return in ? ltx_op_mx4_quantise(c, x, ld, (uint8_t*)q, (uint8_t*)s, n, K, mode, nullptr)
                  : ltx_op_mx4_values(c, (uint8_t*)q, (uint8_t*)s, x, ld, n, K, mode, nullptr);
    };
    for (bool in : {true, false}) {
        for (int mode : {0, 1, 2}) CHECK(rows(in, ptr(0), 256, ptr(1), ptr(2), 7, 256, mode), "%s", ltx_last_error(c));
        fake::log.clear();
        CHECK(rows(in, nullptr, 0, nullptr, nullptr, 0, 256, 0) && launches("") == 0, "%s", ltx_last_error(c));
        for (int K : {0, -128, 64, 129, (1 << 23) + 128}) REFUSED(rows(in, ptr(0), 1 << 24, ptr(1), ptr(2), 7, K, 0), "bad shape");
        REFUSED(rows(in, ptr(0), 256, ptr(1), ptr(2), -1, 256, 0), "bad shape");
        for (int mode : {-1, 3}) REFUSED(rows(in, ptr(0), 256, ptr(1), ptr(2), 7, 256, mode), "unknown mode");
        REFUSED(rows(in, nullptr, 256, ptr(1), ptr(2), 7, 256, 0), "NULL");
        REFUSED(rows(in, ptr(0), 256, nullptr, ptr(2), 7, 256, 0), "NULL");
        REFUSED(rows(in, ptr(0), 256, ptr(1), nullptr, 7, 256, 0), "NULL");
        REFUSED(rows(in, ptr(0) + 8, 256, ptr(1), ptr(2), 7, 256, 0), "16 bytes");
        REFUSED(rows(in, ptr(0), 256, ptr(1) + 8, ptr(2), 7, 256, 0), "16 bytes");
        REFUSED(rows(in, ptr(0), 256, ptr(1), ptr(2) + 2, 7, 256, 0), "on 4");
        for (int64_t ld : {255, 248, 260, -256}) REFUSED(rows(in, ptr(0), ld, ptr(1), ptr(2), 7, 256, 0), "rows of x");
        CHECK(rows(in, ptr(0), 260, ptr(1), ptr(2), 7, 256, 2), "%s", ltx_last_error(c));
        REFUSED(rows(in, ptr(0), 258, ptr(1), ptr(2), 7, 256, 2), "rows of x");
        REFUSED(rows(in, ptr(0), 128, ptr(1), ptr(2), 0x7fffffff, 128, 0), "too many rows");
        REFUSED(rows(in, ptr(0), 1 << 23, ptr(1), ptr(2), 1 << 14, 1 << 23, 0), "too many rows");
    }
    CHECK(!ltx_op_mx4_quantise(nullptr, ptr(0), 128, nullptr, nullptr, 1, 128, 0, nullptr), "NULL context");
    const Linear good{c};
    CHECK(good(), "%s", ltx_last_error(c));
    auto bad = [&](auto set, const char* text) {
        Linear l = good;
        set(l);
        REFUSED(l(), text);
    };
    for (int K : {0, -128, 64, 129}) bad([&](Linear& l) { l.K = K; }, "bad linear shape");
    bad([](Linear& l) { l.M = 0; }, "bad linear shape");
    bad([](Linear& l) { l.N = -1; }, "bad linear shape");
    bad([](Linear& l) { l.mode = 3; }, "unknown mode");
    bad([](Linear& l) { l.mode = 2; }, "mode F32");
    bad([](Linear& l) { l.mode = 2, l.f32 = 1, l.as = nullptr; }, "mode F32");
    bad([](Linear& l) { l.as = nullptr, l.M = 65; }, "64");
    bad([](Linear& l) { l.a = nullptr; }, "NULL");
    bad([](Linear& l) { l.q = nullptr; }, "NULL");
    bad([](Linear& l) { l.s = nullptr; }, "NULL");
    bad([](Linear& l) { l.y = nullptr; }, "NULL");
    bad([](Linear& l) { l.a += 8; }, "16 bytes");
    bad([](Linear& l) { l.q += 4; }, "16 bytes");
    bad([](Linear& l) { l.as += 1; }, "4 bytes");
    bad([](Linear& l) { l.s += 2; }, "4 bytes");
    bad([](Linear& l) { l.bias += 2; }, "aligned");
    bad([](Linear& l) { l.y += 1; }, "aligned");
    bad([](Linear& l) { l.y += 2, l.f32 = 1; }, "aligned");
    bad([](Linear& l) { l.K = (1 << 23) + 128; }, "too many");
    bad([](Linear& l) { l.N = 1 << 21; }, "too many");
    bad([](Linear& l) { l.M = 0x7fffffff; }, "too many");
    bad([](Linear& l) { l.K = 1 << 23, l.N = 1 << 14; }, "too many");
    Linear l = good;
    l.mode = 2, l.f32 = 1;
    CHECK(l(), "%s", ltx_last_error(c));
    l = good;
    l.bias = nullptr, l.y += 2;
    CHECK(l(), "%s", ltx_last_error(c));
    CHECK(!ltx_op_linear_mx4(nullptr, ptr(0), nullptr, nullptr, nullptr, nullptr, nullptr, 0, 1, 1, 128, 0, 0, nullptr), "NULL");
}

// More than 16 rows in values go through scratch of the context, ordered behind its last
// use; a captured call, and one without memory, takes none.
static void mx4_scratch() {
    Linear l{context()};
    ltx_ctx* c = l.c;
    l.as = nullptr, l.M = 40, l.N = 16384, l.K = 4096, l.st = (hipStream_t)0x77;
    fake::log.clear();
    CHECK(l(), "%s", ltx_last_error(c));
    CHECK(launches("ltx_mx4_quantise_f16") == 1 && launches("ltx_gemm_mx4_f16_64k4") == 1 && launches("") == 2, "two launches");
    CHECK(fake::log.back().what == "record", "the scratch's use is recorded");
    uint64_t bytes = 0;
    for (const fake::Op& o : fake::log) bytes += o.what == "malloc" ? o.bytes : 0;
    CHECK(bytes >= 40ull * 4096 * 17 / 32, "%llu", (unsigned long long)bytes);
    fake::log.clear();
    CHECK(l(), "%s", ltx_last_error(c));
    CHECK(fake::log.front().what == "wait", "and waited for");
    l.M = 16;
    fake::log.clear();
    CHECK(l() && fake::log.size() == 1 && launches("ltx_linear_mx4_f16_rows_1_4") == 1, "%s", fake::log.back().name.c_str());
    fake::capturing.insert(l.st);
    for (int M : {17, 33, 64}) {
        l.M = M;
        fake::log.clear();
        CHECK(l() && fake::log.size() == 1 && launches("ltx_linear_mx4_f16_rows_") == 1 && !fake::broken_capture, "%s",
              fake::log.back().name.c_str());
    }
    fake::capturing.clear();
    Linear n{context()};
    n.as = nullptr, n.M = 40;
    fake::limit = fake::in_use;
    fake::log.clear();
    CHECK(n() && launches("ltx_linear_mx4_f16_rows_3_1") == 1 && launches("") == 1, "no memory: %s", fake::log.back().name.c_str());
}

// The kernels that sizes and types select, one a line.
static void kernels() {
    std::set<std::string> names;
    auto take = [&]() {
        for (const fake::Op& o : fake::log)
            if (o.what == "launch") names.insert(o.name);
        fake::log.clear();
    };
    Linear l{context()};
    ltx_ctx* c = l.c;
    for (l.mode = 0; l.mode < 3; l.mode++)
        for (l.f32 = l.mode == 2; l.f32 < 2; l.f32++)
            for (l.gelu = 0; l.gelu < 2; l.gelu++)
                for (const char* as : {(const char*)ptr(1), (const char*)nullptr})
                    for (int captured = 0; captured < 2; captured++)
                        for (int M : {1, 16, 17, 33, 64, 128, 300, 700, 1024, 2970, 28672})
                            for (int N : {1, 64, 2048, 4096, 6144, 8200, 12288, 16400})
                                for (int K : {128, 4096, 16384}) {
                                    if (!as && (M > 64 || l.mode == 2)) continue;
                                    l.as = as, l.M = M, l.N = N, l.K = K;
                                    l.st = captured ? (hipStream_t)0x77 : nullptr;
                                    if (captured) fake::capturing.insert(l.st);
                                    CHECK(l(), "%d %d %d: %s", M, N, K, ltx_last_error(c));
                                    fake::capturing.clear();
                                    take();
                                }
    for (int mode = 0; mode < 3; mode++) {
        CHECK(ltx_op_mx4_quantise(c, ptr(0), 128, (uint8_t*)ptr(1), (uint8_t*)ptr(2), 1, 128, mode, nullptr), "quantise");
        CHECK(ltx_op_mx4_values(c, (uint8_t*)ptr(1), (uint8_t*)ptr(2), ptr(0), 128, 1, 128, mode, nullptr), "values");
        for (int heads : {32, 33, 96})
            for (int norm = 0; norm < 2; norm++) {
                std::vector<double> f(64, 1.0);
                ltx_rope* r = nullptr;
                CHECK(ltx_rope_create(c, 1, 1, f.data(), nullptr, nullptr, &r), "%s", ltx_last_error(c));
                CHECK(ltx_op_qk_rope(c, r, (const double*)ptr(0), 9, ptr(1), 128 * heads, norm ? (const float*)ptr(2) : nullptr,
                                     ptr(3), 128 * heads, heads, nullptr, 0, nullptr, nullptr, 0, 0, 1e-6f, mode, nullptr),
                      "%s", ltx_last_error(c));
                ltx_rope_free(c, r);
            }
        take();
    }
    for (int mode = 0; mode < 2; mode++) {
        ltx_kv_cache* k = nullptr;
        CHECK(ltx_kv_cache_create(c, mode, 8, 100, &k), "%s", ltx_last_error(c));
        for (int rows : {1, 20, 200, 1000, 9000})
            for (int window : {100, 5000, 200000, 9000000}) {
                const ltx_kv_batch b = {1, rows, (const int32_t*)ptr(0), (const int32_t*)ptr(1), (const int32_t*)ptr(2), 200000};
                CHECK(ltx_op_kv_attention_window(c, k, &b, ptr(5), 4096, 32, 1, window, 9, nullptr, ptr(6), 4096, nullptr, 0,
                                                 nullptr),
                      "%s", ltx_last_error(c));
                take();
            }
    }
    for (const std::string& n : names) std::printf("%s\n", n.c_str());
}

// ---- rotary positions -----------------------------------------------------------------

static void rope_refusals() {
    ltx_ctx* c = context();
    std::vector<double> f(4 * 64, 0.5), p(4 * 64, 0.25);
    std::vector<int32_t> x(4 * 64, 1);
    ltx_rope* r = nullptr;
    REFUSED(ltx_rope_create(c, 0, 2, f.data(), nullptr, nullptr, &r), "heads");
    REFUSED(ltx_rope_create(c, 65536, 2, f.data(), nullptr, nullptr, &r), "heads");
    for (int axes : {0, -1, 9}) REFUSED(ltx_rope_create(c, 4, axes, f.data(), nullptr, nullptr, &r), "axes");
    REFUSED(ltx_rope_create(c, 4, 2, nullptr, nullptr, nullptr, &r), "frequencies");
    REFUSED(ltx_rope_create(c, 4, 1, f.data(), p.data(), x.data(), &r), "axis");
    REFUSED(ltx_rope_create(c, 4, 2, f.data(), p.data(), x.data(), nullptr), "NULL");
    for (double bad : {(double)INFINITY, (double)NAN}) {
        auto g = f;
        g[200] = bad;
        REFUSED(ltx_rope_create(c, 4, 2, g.data(), p.data(), x.data(), &r), "finite");
        REFUSED(ltx_rope_create(c, 4, 2, f.data(), g.data(), x.data(), &r), "finite");
    }
    x[70] = -1;
    REFUSED(ltx_rope_create(c, 4, 2, f.data(), p.data(), x.data(), &r), "axis");
    CHECK(!r, "no handle");
    x[70] = 0;
    // beside a capture of another stream, and of the context's own second one
    fake::capturing.insert((hipStream_t)0x77);
    fake::capturing.insert(c->side);
    CHECK(ltx_rope_create(c, 4, 2, f.data(), p.data(), x.data(), &r) && !fake::broken_capture, "%s", ltx_last_error(c));
    ltx_rope* other = nullptr;
    CHECK(ltx_rope_create_grid(c, &other) && !fake::broken_capture, "%s", ltx_last_error(c));
    ltx_rope_free(c, other);
    CHECK(!fake::broken_capture, "the capture is broken");
    fake::capturing.clear();
    ltx_rope_free(c, nullptr);
    struct Call {
        const ltx_rope* r;
        const char *pos = ptr(0), *q = ptr(1), *qn = ptr(2), *k = ptr(4), *kn = ptr(5);
        char *qo = ptr(3), *ko = ptr(6);
        int64_t ldq = 1024, ldqo = 1024, ldk = 512, ldko = 512;
        int rows = 5, heads = 8, kv = 4, mode = 0;
    };
    auto call = [&](const Call& a) {
        return ltx_op_qk_rope(c, a.r, (const double*)a.pos, a.rows, a.q, a.ldq, (const float*)a.qn, a.qo, a.ldqo, a.heads, a.k,
                              a.ldk, (const float*)a.kn, a.ko, a.ldko, a.kv, 1e-6f, a.mode, nullptr);
    };
    const Call good{r};
    CHECK(call(good), "%s", ltx_last_error(c));
    auto bad = [&](auto set, const char* text) {
        Call a = good;
        set(a);
        REFUSED(call(a), text);
    };
    bad([](Call& a) { a.r = nullptr; }, "NULL");
    bad([](Call& a) { a.mode = 4; }, "unknown mode");
    bad([](Call& a) { a.rows = -1; }, "rows");
    for (int heads : {0, -4, 6}) bad([&](Call& a) { a.heads = heads; }, "multiples");
    for (int kv : {0, -4, 6}) bad([&](Call& a) { a.kv = kv; }, "multiples");
    bad([](Call& a) { a.heads = 65536, a.ldq = a.ldqo = 1 << 24; }, "65,535");
    bad([](Call& a) { a.pos = nullptr; }, "positions");
    bad([](Call& a) { a.pos += 4; }, "positions");
    bad([](Call& a) { a.q = nullptr; }, "NULL");
    bad([](Call& a) { a.qo = nullptr; }, "NULL");
    bad([](Call& a) { a.ko = nullptr; }, "NULL");
    bad([](Call& a) { a.q += 8; }, "16 bytes");
    bad([](Call& a) { a.ko += 4; }, "16 bytes");
    bad([](Call& a) { a.ldq = 1016; }, "16 bytes");
    bad([](Call& a) { a.ldqo = 1028; }, "16 bytes");
    bad([](Call& a) { a.ldk = 504; }, "16 bytes");
    bad([](Call& a) { a.qn += 4; }, "weights");
    bad([](Call& a) { a.kn += 8; }, "weights");
    fake::log.clear();
    Call none = good;
    none.rows = 0, none.pos = none.q = nullptr;
    CHECK(call(none) && launches("") == 0, "%s", ltx_last_error(c));
    Call alone = good;
    alone.k = alone.kn = nullptr, alone.ko = nullptr, alone.kv = 77, alone.ldk = 0;
    CHECK(call(alone) && launches("ltx_qk_rope_f16_norm") == 1, "%s", ltx_last_error(c));
    const int live = (int)fake::mem.size();
    ltx_rope_free(c, r);
    CHECK((int)fake::mem.size() == live - 1, "freed");
    fake::limit = fake::in_use;
    r = (ltx_rope*)1;
    CHECK(!ltx_rope_create(c, 4, 2, f.data(), p.data(), x.data(), &r) && !r, "no memory: refused, no handle");
}

// The plan of the blocks: what it turns by is what the tables hold.
static void rope_grid() {
    ltx_ctx* c = context();
    ltx_rope* r = nullptr;
    CHECK(ltx_rope_create_grid(c, &r), "%s", ltx_last_error(c));
    const double* f = (const double*)copied.data();
    const double* p = f + 2048;
    const uint8_t* x = (const uint8_t*)(p + 2048);
    CHECK(copied.size() == 2048 * 17, "%zu", copied.size());
    std::mt19937 rng(5);
    std::uniform_real_distribution<float> u(0, 1);
    for (int trial = 0; trial < 50; trial++) {
        float grid[3][2];
        for (int a = 0; a < 3; a++) {
            grid[a][0] = u(rng) * (a ? 2000 : 19);
            grid[a][1] = grid[a][0] + u(rng);
        }
        std::vector<float> cs(2048), sn(2048);
        CHECK(ltx_rope_tables(&grid[0][0], 1, cs.data(), sn.data(), 1), "%s", ltx_last_error(nullptr));
        for (int j = 0; j < 2048; j++) {
            const double mid = ((double)grid[x[j]][0] + grid[x[j]][1]) / 2, t = (f[j] * mid + p[j]) * M_PI_2;
            CHECK(std::fabs(std::cos(t) - cs[j]) < 1e-7 && std::fabs(std::sin(t) - sn[j]) < 1e-7, "slot %d", j);
        }
    }
}

// ---- windows ----------------------------------------------------------------------------

static void window_refusals() {
    ltx_ctx* c = context();
    ltx_kv_cache* k = nullptr;
    CHECK(ltx_kv_cache_create(c, 0, 8, 100, &k), "%s", ltx_last_error(c));
    ltx_kv_batch b = {3, 10, (const int32_t*)ptr(0), (const int32_t*)ptr(1), (const int32_t*)ptr(2), 4000};
    auto attend = [&](int window, int sinks, void* work = nullptr, uint64_t bytes = 0, int heads = 32, int causal = 1,
                      hipStream_t st = nullptr) {
        return ltx_op_kv_attention_window(c, k, &b, ptr(5), 4096, heads, causal, window, sinks, nullptr, ptr(6), 4096, work,
                                          bytes, st);
    };
    uint64_t n = 0;
    for (int window : {0, -1, (int)0x80000000}) {
        REFUSED(attend(window, 0), "window");
        REFUSED(ltx_op_kv_attention_window_workspace(c, k, &b, 32, 1, window, 0, &n), "window");
    }
    REFUSED(attend(5, -1), "sinks");
    REFUSED(attend(5, 0, nullptr, 0, 12), "heads");
    REFUSED(attend(5, 0, ptr(7) + 8, 1 << 30), "work");
    CHECK(ltx_op_kv_attention_window_workspace(c, k, &b, 32, 1, 9000, 64, &n) && n, "%s", ltx_last_error(c));
    REFUSED(attend(9000, 64, ptr(7), n - 1), "work");
    CHECK(attend(9000, 64, ptr(7), n), "%s", ltx_last_error(c));
    const ltx_kv_batch good = b;
    b.max_pages = 0;
    REFUSED(attend(5, 0), "max_pages");
    b = good;
    b.row_start = (const int32_t*)(ptr(0) + 2);
    REFUSED(attend(5, 0), "4 bytes");
    b = good;
    CHECK(!ltx_op_kv_attention_window(nullptr, k, &b, ptr(5), 4096, 32, 1, 5, 0, nullptr, ptr(6), 4096, nullptr, 0, nullptr),
          "NULL context");
    REFUSED(ltx_op_kv_attention_window(c, nullptr, &b, ptr(5), 4096, 32, 1, 5, 0, nullptr, ptr(6), 4096, nullptr, 0, nullptr),
            "NULL");
    REFUSED(ltx_op_kv_attention_window(c, k, nullptr, ptr(5), 4096, 32, 1, 5, 0, nullptr, ptr(6), 4096, nullptr, 0, nullptr),
            "NULL");
    fake::log.clear();
    b.rows = 0;
    CHECK(attend(5, 0) && launches("") == 0, "%s", ltx_last_error(c));
    b = good;
    // as wide as the table: the kernels without a window
    for (int window : {64 * 4000, 0x7fffffff}) {
        fake::log.clear();
        CHECK(attend(window, 0x7fffffff) && launches("ltx_kv_attn_f16_win") == 0 && launches("ltx_kv_attn_f16") == 1, "%s",
              ltx_last_error(c));
    }
    fake::log.clear();
    CHECK(attend(64 * 4000 - 1, 0x7fffffff) && launches("ltx_kv_attn_f16_win") == 1, "%s", ltx_last_error(c));
    // captured without a workspace: not split
    fake::capturing.insert((hipStream_t)0x77);
    fake::log.clear();
    CHECK(attend(9000, 64, nullptr, 0, 32, 1, (hipStream_t)0x77) && fake::log.size() == 1 && !fake::broken_capture, "%s",
          ltx_last_error(c));
    fake::capturing.clear();
    // one size for calls with row_start and without
    for (int rows : {1, 3, 31, 200})
        for (int window : {10, 2000, 20000}) {
            b = {rows, rows, (const int32_t*)ptr(0), (const int32_t*)ptr(1), (const int32_t*)ptr(2), 448};
            uint64_t with = 0, without = 0;
            CHECK(ltx_op_kv_attention_window_workspace(c, k, &b, 32, 1, window, 70, &with), "%s", ltx_last_error(c));
            b.row_start = nullptr;
            CHECK(ltx_op_kv_attention_window_workspace(c, k, &b, 32, 1, window, 70, &without), "%s", ltx_last_error(c));
            CHECK(with == without && attend(window, 70, with ? ptr(7) : nullptr, with), "%d %d", rows, window);
        }
}

// The pages of a tile's range are those that hold a key some row of it sees, within the
// table, and no more than the sequence's units; with extremes that pass 31 bits.
static void window_index(unsigned seed) {
    std::mt19937 rng(seed);
    auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
    for (int trial = 0; trial < 4000; trial++) {
        const int group = pick(1, 9), tile = 16 << pick(0, 4), causal = pick(0, 1);
        const KvSeq s{0, pick(0, 200), pick(0, 900)};
        const int window = pick(0, 3) ? pick(1, 400) : pick(1, 1 << 30), sinks = pick(0, 2) ? pick(0, 200) : pick(0, 1 << 30);
        const int units = kv_range_units(window, sinks, causal, s, group, tile);
        CHECK(units >= 1 && units <= std::max(1, kv_pages(s.L)), "%d", units);
        for (int t = 0; t < kv_tiles(s.n, group, tile); t++) {
            const KvRange r = kv_tile_range(window, sinks, causal, s, group, t, tile);
            CHECK(r.ps >= 0 && r.skip >= 0 && r.count >= 0 && r.count <= units, "%d %d %d of %d", r.ps, r.skip, r.count, units);
            std::set<int> want, got;
            const int64_t c1 = std::min<int64_t>((int64_t)(t + 1) * tile, (int64_t)s.n * group) - 1;
            bool all = true;
            for (int i = (int)((int64_t)t * tile / group); i <= c1 / group; i++) {
                const int e = kv_limit(causal, s, i);
                all &= e > 0;
                for (int j = 0; j < e; j++)
                    if (j >= (int64_t)e - window || j < sinks) want.insert(j / 64);
            }
            for (int u = 0; u < r.count; u++) got.insert(kv_range_page(r, u));
            for (int page = 0; page <= kv_pages(s.L) + 1; page++) {  // the first u from that page on
                int u = 0;
                while (u < r.count && kv_range_page(r, u) < page) u++;
                const int found = kv_range_find(r, page);
                CHECK(u < r.count ? found == u : found >= r.count, "page %d: %d for %d", page, found, u);
            }
            CHECK((int)got.size() == r.count, "pages twice");
            CHECK(got == want || (!all && std::includes(got.begin(), got.end(), want.begin(), want.end())), "%zu and %zu",
                  got.size(), want.size());
            for (int p : got) CHECK(p >= 0 && p < kv_pages(s.L), "%d", p);
        }
    }
    const KvSeq far{0, 1 << 20, 1 << 30};
    for (int t : {0, 4095}) {
        const KvRange r = kv_tile_range(1 << 30, 1 << 30, 1, far, 1, t, 256);
        CHECK(r.ps == 0 && r.skip == 0 && r.count <= 1 << 24, "%d", r.count);
        const KvRange n = kv_tile_range(1, 0, 1, far, 1, t, 256);
        CHECK(n.count >= 4 && n.count <= 5 && kv_range_page(n, n.count - 1) < 1 << 24, "%d", n.count);
    }
    CHECK(kv_range_units(1 << 30, 1 << 30, 1, far, 1, 256) == 1 << 24, "units");
}

int main(int argc, char** argv) {
    const std::string cmd = argc > 1 ? argv[1] : "";
    if (cmd == "mx4_refusals")
        mx4_refusals();
    else if (cmd == "mx4_scratch")
        mx4_scratch();
    else if (cmd == "kernels")
        kernels();
    else if (cmd == "rope_refusals")
        rope_refusals();
    else if (cmd == "rope_grid")
        rope_grid();
    else if (cmd == "window_refusals")
        window_refusals();
    else if (cmd == "window_index")
        window_index(std::atoi(argv[2]));
    else
        CHECK(false, "unknown command %s", cmd.c_str());
    std::printf("ok\n");
    std::fflush(stdout);
    std::_Exit(0);  // (the library's own teardown belongs to the real runtime)
}
