// The 4-bit cache and linear on the recording HIP stand-in (refusals, workspaces,
// routes), and the kernels' index arithmetic compiled for the host. Run by
// tests/test_kv_host.py.
#include <algorithm>
#include <random>

#include "fake_hip.hpp"
#include "ltx_internal.hpp"
#include "ltx_kv_index.h"

// what fake_hip.hpp leaves out
extern "C" hipError_t hipMemsetAsync(void*, int, size_t, hipStream_t s) {
    return fake::capturing.count(s) ? hipErrorStreamCaptureUnsupported : hipSuccess;
}
static uint64_t counter;      // the count of bad pages, as the device holds it
static uint64_t counted_by_others;  // and what kernels on other streams add right after it is read
extern "C" hipError_t hipMemcpyAsync(void* d, const void* s, size_t n, hipMemcpyKind kind, hipStream_t st) {
    fake::log.push_back({"copy", "", st});
    if (fake::capturing.count(st)) {
        fake::broken_capture = true;
        return hipErrorStreamCaptureUnsupported;
    }
    if (n == 8 && kind == hipMemcpyDeviceToHost) {
        std::memcpy(d, &counter, 8);
        counter += counted_by_others;
    }
    if (n == 8 && kind == hipMemcpyHostToDevice) std::memcpy(&counter, s, 8);
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

struct Fixture {
    ltx_ctx* c = nullptr;
    ltx_kv_cache* cache = nullptr;
    ltx_kv_batch b{};
    Fixture(int heads = 8, int mode = LTX_MODE_F16) {
        CHECK(ltx_init(0, &c), "%s", ltx_last_error(nullptr));
        CHECK(ltx_kv_cache_create(c, mode, heads, 100, &cache), "%s", ltx_last_error(c));
        b = {3, 10, (const int32_t*)ptr(0), (const int32_t*)ptr(1), (const int32_t*)ptr(2), 20};
    }
    int write(const void* k = ptr(3), int64_t ldk = 1024, const void* v = ptr(4), int64_t ldv = 1024) {
        return ltx_op_kv_write(c, cache, &b, k, ldk, v, ldv, nullptr);
    }
    int read(void* k = ptr(3), int64_t ldk = 1024, void* v = ptr(4), int64_t ldv = 1024) {
        return ltx_op_kv_read(c, cache, &b, k, ldk, v, ldv, nullptr);
    }
    int attend(const void* q = ptr(5), int64_t ldq = 4096, int heads = 32, void* out = ptr(6), int64_t ldo = 4096,
               void* work = ptr(7), uint64_t bytes = 1ull << 30, hipStream_t st = nullptr) {
        return ltx_op_kv_attention(c, cache, &b, q, ldq, heads, 1, nullptr, out, ldo, work, bytes, st);
    }
};

#define REFUSED(call, text)                                                                          \
    do {                                                                                             \
        fake::log.clear();                                                                           \
        CHECK(!(call), "taken: %s", #call);                                                          \
        CHECK(std::strstr(ltx_last_error(f.c), text), "%s: %s", #call, ltx_last_error(f.c));         \
        CHECK(launches("") == 0, "%s launched", #call);                                              \
    } while (0)

static void refusals() {
    Fixture f;
    ltx_kv_cache* k = nullptr;
    REFUSED(ltx_kv_cache_create(f.c, LTX_MODE_F32, 8, 10, &k), "16-bit mode");
    REFUSED(ltx_kv_cache_create(f.c, 7, 8, 10, &k), "16-bit mode");
    REFUSED(ltx_kv_cache_create(f.c, 0, 0, 10, &k), "bad cache shape");
    REFUSED(ltx_kv_cache_create(f.c, 0, 8, 0, &k), "bad cache shape");
    REFUSED(ltx_kv_cache_create(f.c, 0, 8, 1 << 25, &k), "at most");
    REFUSED(ltx_kv_cache_create(f.c, 0, 8, 10, nullptr), "NULL");
    CHECK(f.write() && f.read() && f.attend(), "%s", ltx_last_error(f.c));
    REFUSED(ltx_op_kv_write(f.c, nullptr, &f.b, ptr(3), 1024, ptr(4), 1024, nullptr), "NULL");
    REFUSED(ltx_op_kv_write(f.c, f.cache, nullptr, ptr(3), 1024, ptr(4), 1024, nullptr), "NULL");
    CHECK(!ltx_op_kv_write(nullptr, f.cache, &f.b, ptr(3), 1024, ptr(4), 1024, nullptr), "NULL context");
    CHECK(!ltx_op_kv_attention(nullptr, f.cache, &f.b, ptr(3), 4096, 32, 1, nullptr, ptr(4), 4096, nullptr, 0, nullptr),
          "NULL context");
    const ltx_kv_batch good = f.b;
    auto each = [&](auto set, const char* text) {
        f.b = good;
        set(f.b);
        REFUSED(f.write(), text);
        REFUSED(f.read(), text);
        REFUSED(f.attend(), text);
        uint64_t n;
        REFUSED(ltx_op_kv_attention_workspace(f.c, f.cache, &f.b, 32, &n), text);
        f.b = good;
    };
    each([](ltx_kv_batch& b) { b.nseq = 0; }, "nseq");
    each([](ltx_kv_batch& b) { b.rows = -1; }, "rows");
    each([](ltx_kv_batch& b) { b.max_pages = 0; }, "max_pages");
    each([](ltx_kv_batch& b) { b.max_pages = (1 << 24) + 1; }, "max_pages");
    each([](ltx_kv_batch& b) { b.kv_len = nullptr; }, "kv_len");
    each([](ltx_kv_batch& b) { b.pages = nullptr; }, "pages");
    each([](ltx_kv_batch& b) { b.row_start = nullptr; }, "row_start");
    REFUSED(f.write(nullptr), "k is NULL");
    REFUSED(f.write(ptr(3) + 8), "k:");
    REFUSED(f.write(ptr(3), 1023), "k:");
    REFUSED(f.write(ptr(3), 1016), "k:");
    REFUSED(f.write(ptr(3), 1028), "k:");
    REFUSED(f.write(ptr(3), 1024, nullptr), "v is NULL");
    REFUSED(f.write(ptr(3), 1024, ptr(4), 8), "v:");
    REFUSED(f.read(ptr(3), 1024, ptr(4) + 2), "v:");
    REFUSED(f.attend(nullptr), "q is NULL");
    REFUSED(f.attend(ptr(5), 4088), "q:");
    REFUSED(f.attend(ptr(5), 4096, 32, ptr(6) + 4), "out:");
    REFUSED(f.attend(ptr(5), 4096, 0), "heads");
    REFUSED(f.attend(ptr(5), 4096, 12), "heads");
    REFUSED(f.attend(ptr(5), 4096, 32, ptr(6), 4096, ptr(7) + 8), "work");
    uint64_t n = 0;
    CHECK(ltx_op_kv_attention_workspace(f.c, f.cache, &f.b, 32, &n) && n, "%s", ltx_last_error(f.c));
    REFUSED(f.attend(ptr(5), 4096, 32, ptr(6), 4096, ptr(7), n - 1), "work");
    CHECK(f.attend(ptr(5), 4096, 32, ptr(6), 4096, ptr(7), n), "%s", ltx_last_error(f.c));
    // no rows: nothing to do, nothing launched
    fake::log.clear();
    f.b.rows = 0;
    CHECK(f.write() && f.read() && f.attend() && launches("") == 0, "%s", ltx_last_error(f.c));
    f.b.rows = 1 << 24;
    REFUSED(f.attend(), "too many rows");
    f.b.rows = 1 << 28;
    REFUSED(f.write(), "too many rows");
    REFUSED(f.read(), "too many rows");

    auto q4 = [&](const void* a, const void* q, const void* s, int s16, const void* bias, void* y, int f32, int M, int N,
                  int K, int mode) {
        return ltx_op_linear_q4(f.c, a, (const uint8_t*)q, s, s16, (const float*)bias, y, f32, M, N, K, 0, mode, nullptr);
    };
    CHECK(q4(ptr(0), ptr(1), ptr(2), 1, ptr(3), ptr(4), 0, 5, 33, 128, 0), "%s", ltx_last_error(f.c));
    for (int bad : {0, -1, 64, 129, 130})
        REFUSED(q4(ptr(0), ptr(1), ptr(2), 1, ptr(3), ptr(4), 0, 5, 32, bad, 0), "bad linear shape");
    REFUSED(q4(ptr(0), ptr(1), ptr(2), 1, ptr(3), ptr(4), 0, 0, 32, 128, 0), "bad linear shape");
    REFUSED(q4(ptr(0), ptr(1), ptr(2), 1, ptr(3), ptr(4), 0, 5, -3, 128, 0), "bad linear shape");
    REFUSED(q4(ptr(0), ptr(1), ptr(2), 1, ptr(3), ptr(4), 0, 5, 32, 128, 3), "unknown mode");
    REFUSED(q4(ptr(0), ptr(1), ptr(2), 1, ptr(3), ptr(4), 0, 5, 32, 128, 2), "f32 output");
    REFUSED(q4(ptr(0) + 8, ptr(1), ptr(2), 1, ptr(3), ptr(4), 0, 5, 32, 128, 0), "16 bytes");
    REFUSED(q4(ptr(0), ptr(1) + 4, ptr(2), 1, ptr(3), ptr(4), 0, 5, 32, 128, 0), "16 bytes");
    REFUSED(q4(ptr(0), ptr(1), ptr(2) + 2, 0, ptr(3), ptr(4), 0, 5, 32, 128, 0), "scales");
    REFUSED(q4(ptr(0), ptr(1), ptr(2), 1, ptr(3) + 2, ptr(4), 0, 5, 32, 128, 0), "bias");
    REFUSED(q4(ptr(0), ptr(1), ptr(2), 1, ptr(3), ptr(4) + 2, 1, 5, 32, 128, 0), "y");
    REFUSED(q4(nullptr, ptr(1), ptr(2), 1, ptr(3), ptr(4), 1, 5, 32, 128, 0), "NULL");
    REFUSED(q4(ptr(0), ptr(1), ptr(2), 1, ptr(3), ptr(4), 0, 1 << 21, 32, 128, 0), "too many rows");
    REFUSED(q4(ptr(0), ptr(1), ptr(2), 1, ptr(3), ptr(4), 0, 1, 1 << 27, 128, 0), "too many rows");
    REFUSED(q4(ptr(0), ptr(1), ptr(2), 1, ptr(3), ptr(4), 0, 1, 32, (1 << 23) + 128, 0), "too many rows");
}

// Without `work`: scratch of the context, ordered behind its last use; a captured
// call, and one without memory, runs unsplit and needs none.
static void scratch() {
    Fixture f;
    hipStream_t s = (hipStream_t)0x77;
    fake::log.clear();
    CHECK(f.attend(ptr(5), 4096, 32, ptr(6), 4096, nullptr, 0, s), "%s", ltx_last_error(f.c));
    CHECK(launches("ltx_kv_attn") == 1 && launches("ltx_kv_join") == 1, "split");
    CHECK(fake::log.back().what == "record", "the scratch's use is recorded");
    fake::log.clear();
    CHECK(f.attend(ptr(5), 4096, 32, ptr(6), 4096, nullptr, 0, s), "%s", ltx_last_error(f.c));
    CHECK(fake::log.front().what == "wait", "and waited for");
    fake::log.clear();
    fake::capturing.insert(s);
    CHECK(f.attend(ptr(5), 4096, 32, ptr(6), 4096, nullptr, 0, s), "%s", ltx_last_error(f.c));
    CHECK(fake::log.size() == 1 && launches("ltx_kv_attn") == 1 && !fake::broken_capture, "captured: one launch");
    fake::log.clear();
    CHECK(f.attend(ptr(5), 4096, 32, ptr(6), 4096, ptr(7), 1ull << 30, s), "%s", ltx_last_error(f.c));
    CHECK(launches("ltx_kv_attn") == 1 && launches("ltx_kv_join") == 1 && fake::log.size() == 2, "captured with work");
    fake::capturing.clear();
    Fixture g;
    fake::limit = fake::in_use;
    fake::log.clear();
    CHECK(g.attend(ptr(5), 4096, 32, ptr(6), 4096, nullptr, 0, s), "%s", ltx_last_error(g.c));
    CHECK(launches("ltx_kv_attn") == 1 && launches("ltx_kv_join") == 0, "no memory: not split");
}

static void memory() {
    const uint64_t before = fake::in_use;
    Fixture f;
    const uint64_t with = fake::in_use;
    CHECK(ltx_kv_cache_bytes(f.cache) >= 100ull * 64 * 8 * 136, "%llu", (unsigned long long)ltx_kv_cache_bytes(f.cache));
    ltx_kv_cache_free(f.c, f.cache);
    CHECK(with - fake::in_use >= 100ull * 64 * 8 * 136 && before <= fake::in_use, "freed");
    // made and freed beside a capture of another stream, in the global mode
    fake::capturing.insert((hipStream_t)0x77);
    ltx_kv_cache* beside = nullptr;
    CHECK(ltx_kv_cache_create(f.c, 0, 8, 100, &beside), "%s", ltx_last_error(f.c));
    ltx_kv_cache_free(f.c, beside);
    CHECK(!fake::broken_capture, "the capture is broken");
    fake::capturing.clear();
    fake::limit = fake::in_use;
    ltx_kv_cache* k = (ltx_kv_cache*)1;
    CHECK(!ltx_kv_cache_create(f.c, 0, 8, 100, &k) && !k, "no memory: refused, no handle");
    ltx_kv_cache_free(f.c, nullptr);
}

// Made while a forward of the same context is being captured, whose second stream
// the capture holds.
static void own_capture() {
    Fixture f;
    fake::capturing.insert((hipStream_t)0x77);
    fake::capturing.insert(f.c->side);
    ltx_kv_cache* k = nullptr;
    CHECK(ltx_kv_cache_create(f.c, 0, 8, 100, &k), "%s", ltx_last_error(f.c));
    ltx_kv_cache_free(f.c, k);
    CHECK(!fake::broken_capture, "the capture is broken");
    for (const fake::Op& o : fake::log) CHECK(!o.stream || !fake::capturing.count(o.stream), "%s", o.what.c_str());
    fake::capturing.clear();
}

// The count of bad pages beside a capture: read on the stream that is named, refused
// on one that is being captured, and the capture is whole.
static void faults_beside_a_capture() {
    Fixture f;
    hipStream_t captured = (hipStream_t)0x77, other = (hipStream_t)0x55;
    fake::capturing.insert(captured);
    counter = 5;
    uint64_t n = 0;
    CHECK(ltx_kv_cache_faults(f.c, f.cache, other, &n, 0) && n == 5, "%s", ltx_last_error(f.c));
    CHECK(!fake::broken_capture, "the capture is broken");
    REFUSED(ltx_kv_cache_faults(f.c, f.cache, captured, &n, 1), "captured");
    CHECK(fake::log.empty() && !fake::broken_capture && counter == 5, "the capture is broken");
    fake::capturing.clear();
    CHECK(ltx_kv_cache_faults(f.c, f.cache, captured, &n, 1) && n == 5, "%s", ltx_last_error(f.c));
    CHECK(ltx_kv_cache_faults(f.c, f.cache, captured, &n, 1) && n == 0, "%s", ltx_last_error(f.c));
}

// Nothing is lost between a reading and its reset, nor to other streams' kernels that
// count meanwhile.
static void faults_are_not_lost() {
    Fixture f;
    uint64_t n = 0, all = 0;
    counter = 7;
    counted_by_others = 3;
    for (int i = 0; i < 4; i++) {
        CHECK(ltx_kv_cache_faults(f.c, f.cache, nullptr, &n, 1) && n == (i ? 3u : 7u), "%llu", (unsigned long long)n);
        all += n;
    }
    counted_by_others = 0;
    for (int reset = 0; reset < 2; reset++)
        CHECK(ltx_kv_cache_faults(f.c, f.cache, nullptr, &n, reset) && n == 3, "%llu", (unsigned long long)n);
    CHECK(all + n == counter && ltx_kv_cache_faults(f.c, f.cache, nullptr, &n, 1) && n == 0, "%llu", (unsigned long long)n);
}

// A workspace's size serves calls with row_start and without.
static void workspace_forms() {
    int split = 0;
    for (int heads : {32, 8, 4, 3})
        for (int group : {1, 4, 20}) {
            Fixture f(heads);
            for (int n : {1, 3, 16, 31, 70, 200})
                for (int width : {1, 20, 128, 448}) {
                    f.b = {n, n, (const int32_t*)ptr(0), (const int32_t*)ptr(1), (const int32_t*)ptr(2), width};
                    ltx_kv_batch one = f.b;
                    one.row_start = nullptr;
                    uint64_t with = 0, without = 0;
                    CHECK(ltx_op_kv_attention_workspace(f.c, f.cache, &f.b, heads * group, &with), "%s", ltx_last_error(f.c));
                    CHECK(ltx_op_kv_attention_workspace(f.c, f.cache, &one, heads * group, &without), "%s", ltx_last_error(f.c));
                    split += with > 0;
                    const int64_t ld = heads * group * 128;
                    auto taken = [&](uint64_t bytes) {
                        return f.attend(ptr(5), ld, heads * group, ptr(6), ld, bytes ? ptr(7) : nullptr, bytes);
                    };
                    CHECK(with == without && taken(without), "%d of %d, %d heads x %d, %d pages: %s", n, n, heads, group,
                          width, ltx_last_error(f.c));
                    f.b = one;
                    CHECK(taken(with), "%s", ltx_last_error(f.c));
                }
        }
    CHECK(split > 50, "%d", split);
}

// A call that cannot split (captured, no workspace) does not take the 256-column tiles
// that only a split makes worth while: few workgroups would walk all pages. Where such
// tiles fill the CUs by themselves, it does.
static void unsplit_tiles() {
    Fixture f;
    hipStream_t s = (hipStream_t)0x77;
    auto kernel = [&](bool captured, int rows, int pages) {
        f.b = {1, rows, (const int32_t*)ptr(0), (const int32_t*)ptr(1), (const int32_t*)ptr(2), pages};
        if (captured) fake::capturing.insert(s);
        fake::log.clear();
        CHECK(f.attend(ptr(5), 4096, 32, ptr(6), 4096, nullptr, 0, s), "%s", ltx_last_error(f.c));
        fake::capturing.clear();
        for (const fake::Op& o : fake::log)
            if (o.what == "launch") return o.name;
        return std::string();
    };
    CHECK(kernel(false, 256, 448) == "ltx_kv_attn_f16_rows2_split", "%s", kernel(false, 256, 448).c_str());
    CHECK(kernel(true, 256, 448) == "ltx_kv_attn_f16", "%s", kernel(true, 256, 448).c_str());
    CHECK(kernel(false, 1024, 448) == "ltx_kv_attn_f16_rows2_split", "%s", kernel(false, 1024, 448).c_str());
    CHECK(kernel(true, 1024, 448) == "ltx_kv_attn_f16_rows1", "%s", kernel(true, 1024, 448).c_str());
    for (bool captured : {false, true})
        CHECK(kernel(captured, 4096, 448) == "ltx_kv_attn_f16_rows2", "%s", kernel(captured, 4096, 448).c_str());
}

// The largest count of rows written or read: 16 a workgroup of 256 threads, fewer than
// 2^32 threads.
static void row_limit() {
    Fixture f;
    for (int rows : {0x0fffffff, (1 << 28) - 15}) {
        f.b.rows = rows;
        REFUSED(f.write(), "too many rows");
        REFUSED(f.read(), "too many rows");
    }
    f.b.rows = (1 << 28) - 16;
    CHECK(f.write() && f.read(), "%s", ltx_last_error(f.c));
}

// Arrays that do not start on their type are refused: the kernels' scalar loads take the
// address without its last two bits.
static void alignment() {
    Fixture f;
    const ltx_kv_batch good = f.b;
    uint64_t n;
    for (int i = 0; i < 3; i++)
        for (int off = 1; off < 4; off++) {
            f.b = good;
            const int32_t*& p = i == 0 ? f.b.row_start : i == 1 ? f.b.kv_len : f.b.pages;
            p = (const int32_t*)((char*)p + off);
            REFUSED(f.write(), "4 bytes");
            REFUSED(f.read(), "4 bytes");
            REFUSED(f.attend(), "4 bytes");
            REFUSED(ltx_op_kv_attention_workspace(f.c, f.cache, &f.b, 32, &n), "4 bytes");
        }
    f.b = good;
    for (int off = 0; off < 4; off++) {
        auto call = [&]() {
            return ltx_op_kv_attention(f.c, f.cache, &f.b, ptr(5), 4096, 32, 1, (const float*)(ptr(8) + off), ptr(6), 4096,
                                       ptr(7), 1ull << 30, nullptr);
        };
        if (off)
            REFUSED(call(), "4 bytes");
        else
            CHECK(call(), "%s", ltx_last_error(f.c));
    }
}

// Every tile form of the linear is one that sizes select: rows and columns of
// test_gpu_q4_forms.py's sweep.
static void linear_forms() {
    Fixture f;
    std::set<std::string> names;
    for (int mode : {LTX_MODE_F16, LTX_MODE_BF16, LTX_MODE_F32})
        for (int s16 : {0, 1})
            for (int N : {48, 4112, 8200, 16400})
                for (int M : {1, 3, 5, 16, 17, 32, 33, 64}) {
                    fake::log.clear();
                    CHECK(ltx_op_linear_q4(f.c, ptr(0), (const uint8_t*)ptr(1), ptr(2), s16, nullptr, ptr(4), 1, M, N, 4736, 0,
                                           mode, nullptr),
                          "%s", ltx_last_error(f.c));
                    CHECK(fake::log.size() == 1, "%zu", fake::log.size());
                    names.insert(fake::log[0].name);
                }
    for (const char* form : {"f16", "bf16", "f32", "f32p"})
        for (const char* scale : {"s16", "s32"})
            for (int mt : {1, 2})
                for (int nt : {1, 2, 4}) {
                    if (mt == 2 && form[0] == 'f' && form[1] == '3') continue;  // mode F32: 16 rows
                    const std::string name = std::string("ltx_linear_q4_") + form + "_" + scale + "_" + std::to_string(mt) +
                                             "_" + std::to_string(nt);
                    CHECK(names.erase(name) == 1, "%s", name.c_str());
                }
    CHECK(names.empty(), "%s", names.begin()->c_str());
}

// The index arithmetic on arrays of any contents: what a kernel would read and
// write stays inside what the call names, and the items fit the grid.
static void index_bounds(unsigned seed) {
    std::mt19937 rng(seed);
    auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
    const int wild[] = {0, 1, -1, 63, 64, 65, 0x7fffffff, (int)0x80000000, 100, 1 << 24};
    for (int trial = 0; trial < 2000; trial++) {
        const bool sane = trial % 2 == 0;
        const int nseq = pick(1, 9), max_pages = pick(1, 12), pool = pick(1, 30), group = pick(1, 9);
        const int tile = 16 << pick(0, 4), slots = pick(1, 40), least = pick(1, 8);
        int rows = pick(0, 90);
        std::vector<int32_t> start(nseq + 1), len(nseq), pages(nseq * max_pages);
        for (auto& p : pages) p = pick(0, 3) ? pick(0, pool - 1) : wild[pick(0, 9)];
        for (int b = 0; b < nseq; b++) len[b] = sane ? pick(0, 64 * max_pages) : wild[pick(0, 9)];
        if (sane) {
            for (auto& s : start) s = pick(0, rows);
            std::sort(start.begin(), start.end());
            start[0] = 0;
        } else
            for (auto& s : start) s = pick(0, 1) ? pick(-5, rows + 5) : wild[pick(0, 9)];
        LtxKvBatchArgs a{nullptr, nullptr, nullptr, start.data(), len.data(), pages.data(), nseq, rows, max_pages, pool, 3};
        for (int b = 0; b < nseq; b++) {
            const KvSeq s = kv_seq(a, b);
            CHECK(s.s0 >= 0 && s.n >= 0 && s.s0 + s.n <= rows && s.L >= 0 && s.L <= 64 * max_pages, "%d %d %d", s.s0, s.n, s.L);
            for (int row = -1; row <= rows; row++) {
                const int pos = kv_position(s, row);
                CHECK(pos == -1 || (pos >= 0 && pos / 64 < max_pages && row >= s.s0 && row < s.s0 + s.n), "%d", pos);
                if (pos < 0) continue;
                const int page = kv_page(a, b, pos / 64);
                CHECK(kv_in_pool(a, page) == (page >= 0 && page < pool), "%d", page);
                CHECK(kv_limit(1, s, row - s.s0) == pos + 1, "%d", pos);
            }
        }
        // the split: items of `per` units over the tiles in order; every unit once, every
        // partial result at a place of its own below the count that the host sizes
        const int64_t bound = (int64_t)rows * group / tile + nseq;
        std::vector<int> pages_of;
        uint32_t units = 0;
        for (int b = 0; b < nseq; b++) {
            const KvSeq s = kv_seq(a, b);
            const int tiles = kv_tiles(s.n, group, tile);
            for (int t = 0; t < tiles; t++) {
                for (int causal = 0; causal < 2; causal++) {
                    const int limit = kv_tile_limit(causal, s, group, t, tile);
                    CHECK(limit >= 0 && limit <= s.L && kv_pages(limit) <= kv_units(s.L), "%d of %d", limit, s.L);
                }
                pages_of.push_back(kv_units(s.L));
                units += kv_units(s.L);
            }
        }
        if (sane) CHECK((int64_t)pages_of.size() <= bound, "%zu tiles", pages_of.size());
        const int per = kv_per_of(units, slots, least);
        CHECK(per >= least && (int64_t)per * slots >= units, "%d", per);
        int last = -1;
        uint32_t at = 0;
        for (int e = 0; e < (int)pages_of.size(); e++) {
            const uint32_t i0 = at / per, i1 = (at + pages_of[e] - 1) / per;
            CHECK(i1 < (uint32_t)slots && (int)(i0 + e) > last, "item %u for tile %d", i0, e);
            last = (int)(i1 + e);
            if (sane) CHECK(last < slots + bound, "part %d", last);
            at += pages_of[e];
        }
    }
    LtxKvBatchArgs big{nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 1, 1, 1, 1 << 25, 32};
    CHECK(kv_block(big, (1 << 25) - 1, 31) == ((1ull << 30) - 1) * LTX_KV_BLOCK, "places pass 32 bits");
}

int main(int argc, char** argv) {
    const std::string cmd = argc > 1 ? argv[1] : "";
    if (cmd == "refusals")
        refusals();
    else if (cmd == "scratch")
        scratch();
    else if (cmd == "memory")
        memory();
    else if (cmd == "own_capture")
        own_capture();
    else if (cmd == "faults_beside_a_capture")
        faults_beside_a_capture();
    else if (cmd == "faults_are_not_lost")
        faults_are_not_lost();
    else if (cmd == "workspace_forms")
        workspace_forms();
    else if (cmd == "unsplit_tiles")
        unsplit_tiles();
    else if (cmd == "row_limit")
        row_limit();
    else if (cmd == "alignment")
        alignment();
    else if (cmd == "linear_forms")
        linear_forms();
    else if (cmd == "index")
        index_bounds(std::atoi(argv[2]));
    else
        CHECK(false, "unknown command %s", cmd.c_str());
    std::printf("ok\n");
    std::fflush(stdout);
    std::_Exit(0);  // (the library's own teardown belongs to the real runtime)
}
