// nt_call_packed: the generation step's entry points with their arguments in one
// array.  A ctypes call converts each of two dozen arguments for ~0.08 us; packing
// them takes 0.2 us together, which a call of 10 us notices.
#include "nt_common.cuh"

#include <cstring>

using namespace nt;

namespace {

// Reads the words in order.
struct Words {
    const char* p;
    int64_t i() {
        int64_t v;
        memcpy(&v, p, 8);
        p += 8;
        return v;
    }
    double d() {
        double v;
        memcpy(&v, p, 8);
        p += 8;
        return v;
    }
    float f() { return (float)d(); }
    template <typename T> T* ptr() { return reinterpret_cast<T*>(static_cast<uintptr_t>(i())); }
};

constexpr int64_t kWords[4] = {21, 25, 27, 27};

}  // namespace

extern "C" int nt_call_packed(int entry, const void* words, int64_t n_words) {
    if (entry < 0 || entry > 3) return fail(NT_ERR_ARG, "nt_call_packed: entry %d", entry);
    if (!words) return fail(NT_ERR_ARG, "nt_call_packed: null pointer");
    if (n_words != kWords[entry])
        return fail(NT_ERR_ARG, "nt_call_packed: %lld words for entry %d, which takes %lld", (long long)n_words, entry,
                    (long long)kWords[entry]);
    Words w{static_cast<const char*>(words)};
    // one variable per argument: the order in which a call's arguments are evaluated is not fixed
    if (entry == NT_ENTRY_ROTARY) {
        const int64_t dtype = w.i(), B = w.i(), T = w.i(), H = w.i(), D = w.i(), R = w.i(), inter = w.i(), inverse = w.i();
        const float mscale = w.f();
        const void* x = w.ptr<void>();
        const int64_t x_sb = w.i(), x_st = w.i(), x_sh = w.i();
        const int64_t* pos = w.ptr<int64_t>();
        const int64_t p_sb = w.i();
        const float* freq = w.ptr<float>();
        void* y = w.ptr<void>();
        const int64_t y_sb = w.i(), y_st = w.i(), y_sh = w.i();
        return nt_rotary((int)dtype, B, T, H, D, R, (int)inter, (int)inverse, mscale, x, x_sb, x_st, x_sh, pos, p_sb, freq, y,
                         y_sb, y_st, y_sh, w.ptr<void>());
    }
    if (entry == NT_ENTRY_KV_APPEND) {
        const int64_t dtype = w.i(), B = w.i(), T = w.i(), H = w.i(), D = w.i(), page = w.i(), pages = w.i(), blocks = w.i();
        const void* k = w.ptr<void>();
        const int64_t k_sb = w.i(), k_st = w.i(), k_sh = w.i();
        const void* v = w.ptr<void>();
        const int64_t v_sb = w.i(), v_st = w.i(), v_sh = w.i();
        void* kc = w.ptr<void>();
        float* ks = w.ptr<float>();
        void* vc = w.ptr<void>();
        float* vs = w.ptr<float>();
        const int32_t* table = w.ptr<int32_t>();
        const int64_t table_sb = w.i();
        const int32_t* lengths = w.ptr<int32_t>();
        const int32_t* counts = w.ptr<int32_t>();
        return nt_kv_append((int)dtype, B, T, H, D, page, pages, blocks, k, k_sb, k_st, k_sh, v, v_sb, v_st, v_sh, kc, ks, vc,
                            vs, table, table_sb, lengths, counts, w.ptr<void>());
    }
    if (entry == NT_ENTRY_KV_ATTENTION) {
        const int64_t dtype = w.i(), B = w.i(), T = w.i(), Hq = w.i(), H = w.i(), D = w.i(), page = w.i(), pages = w.i(),
                      blocks = w.i(), window = w.i();
        const float scale = w.f();
        const void* q = w.ptr<void>();
        const int64_t q_sb = w.i(), q_st = w.i(), q_sh = w.i();
        const void* kc = w.ptr<void>();
        const float* ks = w.ptr<float>();
        const void* vc = w.ptr<void>();
        const float* vs = w.ptr<float>();
        const int32_t* table = w.ptr<int32_t>();
        const int64_t table_sb = w.i();
        const int32_t* lengths = w.ptr<int32_t>();
        const int32_t* counts = w.ptr<int32_t>();
        void* out = w.ptr<void>();
        void* ws = w.ptr<void>();
        const int64_t bytes = w.i();
        return nt_kv_attention((int)dtype, B, T, Hq, H, D, page, pages, blocks, window, scale, q, q_sb, q_st, q_sh, kc, ks, vc,
                               vs, table, table_sb, lengths, counts, out, ws, bytes, w.ptr<void>());
    }
    const int64_t dtype = w.i(), B = w.i(), V = w.i();
    const void* x = w.ptr<void>();
    const int64_t ld = w.i();
    const int64_t* tokens = w.ptr<int64_t>();
    const int64_t tok_ld = w.i(), L = w.i();
    const int32_t* lengths = w.ptr<int32_t>();
    const int32_t* prompts = w.ptr<int32_t>();
    const int64_t each = w.i();
    const float* rep = w.ptr<float>();
    const double rep_all = w.d();
    const float* freq = w.ptr<float>();
    const float freq_all = w.f();
    const float* pres = w.ptr<float>();
    const float pres_all = w.f();
    const int64_t* ids = w.ptr<int64_t>();
    const int64_t ids_ld = w.i();
    const float* bias = w.ptr<float>();
    const int64_t bias_ld = w.i(), NB = w.i();
    const uint32_t* allowed = w.ptr<uint32_t>();
    const int64_t allowed_ld = w.i();
    void* out = w.ptr<void>();
    const int64_t ldo = w.i();
    return nt_logits_process((int)dtype, B, V, x, ld, tokens, tok_ld, L, lengths, prompts, (int)each, rep, rep_all, freq,
                             freq_all, pres, pres_all, ids, ids_ld, bias, bias_ld, NB, allowed, allowed_ld, out, ldo,
                             w.ptr<void>());
}
