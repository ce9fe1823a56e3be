// Calls the sequence operators' XLA handlers with buffers of the host, whose addresses nothing reads: the C entry points here only write down
// what they were given. `handlers` prints a line for each case: its name, then "called" and the descriptors or "refused" and the message.
#define CCK_FFI
#include "ffi_handler.cu"

#include <cstdio>
#include <map>
#include <sstream>

static std::string g_seen; // what the last entry point was given

static std::string text(const cck_rows* r) {
    std::ostringstream o;
    o << " rows(" << r->heads << " " << r->row_stride << " " << r->head_stride << " " << r->dtype << ")";
    return o.str();
}
static std::string text(const cck_rotation* r) {
    std::ostringstream o;
    o << " rotation(" << r->dims << " " << r->axes << " " << r->adjacent << " " << r->section[0] << " " << r->section[1] << " " << r->pos_stride << ")";
    return o.str();
}
static std::string text(const cck_cache* c) {
    std::ostringstream o;
    o << " cache(" << c->pages << " " << c->page_tokens << " " << c->heads << " " << c->dim << ")";
    return o.str();
}
static std::string text(const cck_batch* b) {
    std::ostringstream o;
    o << " batch(" << b->sequences << " " << b->rows << " " << b->max_new << " " << b->max_len << " " << b->table_pages << " " << b->table_stride << ")";
    return o.str();
}
extern "C" {
int cck_mk_sample(void*, const int*, const void* const*, const size_t*, int, float*, int, void*, size_t, int, int, int) {
    return CCK_OK;
}
const char* cck_last_error() {
    return "";
}
int cck_rotary(void*, const cck_rotation* r, int rows, int dim, const cck_rows* x, const cck_rows* y, int inverse) {
    g_seen = text(r) + " " + std::to_string(rows) + " " + std::to_string(dim) + text(x) + text(y) + " " + std::to_string(inverse);
    return CCK_OK;
}
int cck_cache_append(void*, const cck_cache* c, const cck_batch* b, const cck_rows* k, const cck_rows* v, const cck_rotation* r, const cck_rows* q, const cck_rows* out, int32_t*) {
    g_seen = text(c) + text(b) + text(k) + text(v) + text(r) + text(q) + text(out);
    return CCK_OK;
}
int cck_cache_attention(void*, const cck_cache* c, const cck_batch* b, const cck_rows* q, const cck_rows* out, float*, float scale, int causal, int window, void*, size_t ws) {
    g_seen = text(c) + text(b) + text(q) + text(out) + " " + std::to_string(scale) + " " + std::to_string(causal) + " " + std::to_string(window) + " " + std::to_string(ws);
    return CCK_OK;
}
}

using ffi::AnyBuffer;
using D = ffi::DataType;
using Buffers = std::map<std::string, AnyBuffer>;
static char g_memory[64];

static AnyBuffer buffer(D type, std::vector<int64_t> dims, int at = 0) {
    AnyBuffer b;
    b.data = g_memory + at, b.type = type, b.dims = std::move(dims);
    return b;
}
// six rows of 4 query heads and 2 heads of the cache of 64, 3 sequences, 10 pages of 16 tokens
static Buffers good() {
    return {
        {"x", buffer(D::BF16, {6, 4, 64})}, {"y", buffer(D::BF16, {6, 4, 64})}, {"q", buffer(D::BF16, {6, 4, 64})}, {"out", buffer(D::BF16, {6, 4, 64})},
        {"k", buffer(D::BF16, {6, 2, 64})}, {"v", buffer(D::BF16, {6, 2, 64})}, {"freq", buffer(D::F32, {32})}, {"pos", buffer(D::S32, {2, 6})},
        {"kc", buffer(D::F8E4M3FN, {10, 2, 16, 64})}, {"vc", buffer(D::U8, {10 * 2 * 16 * 64}, 1)}, {"ks", buffer(D::F32, {10, 2}, 2)}, {"vs", buffer(D::F32, {10, 2}, 3)},
        {"kc_out", buffer(D::F8E4M3FN, {10, 2, 16, 64})}, {"vc_out", buffer(D::U8, {10 * 2 * 16 * 64}, 1)}, {"ks_out", buffer(D::F32, {10, 2}, 2)},
        {"vs_out", buffer(D::F32, {10, 2}, 3)}, {"first", buffer(D::S32, {4})}, {"len", buffer(D::S32, {3})}, {"table", buffer(D::S32, {3, 5})},
        {"lse", buffer(D::F32, {6, 4})}, {"ws", buffer(D::U8, {4096})},
    };
}
static ffi::Error call(const std::string& target, Buffers& b, std::vector<int64_t> section) {
    auto out = [&](const char* n) { return ffi::Result<AnyBuffer>{b[n]}; };
    if (target == "rotary") {
        return rotary_ffi(nullptr, b["x"], b["freq"], b["pos"], out("y"), {section}, 1, 1);
    }
    if (target == "append") {
        return cache_append_ffi(nullptr, b["kc"], b["vc"], b["ks"], b["vs"], b["k"], b["v"], b["q"], b["freq"], b["pos"], b["first"], b["len"], b["table"], out("kc_out"),
                                out("vc_out"), out("ks_out"), out("vs_out"), out("out"), {section}, 0, 16, 3, 70);
    }
    return cache_attention_ffi(nullptr, b["kc"], b["vc"], b["ks"], b["vs"], b["q"], b["first"], b["len"], b["table"], out("out"), out("lse"), out("ws"), 0.125f, 1, 7, 16, 3, 70);
}

static D type_of(const std::string& s) {
    const std::map<std::string, D> all = {{"bf16", D::BF16}, {"f16", D::F16}, {"f32", D::F32}, {"f64", D::F64}, {"f8", D::F8E4M3FN}, {"s8", D::S8}, {"u8", D::U8}, {"s32", D::S32}, {"s64", D::S64}};
    return all.at(s);
}

// arguments, in threes: target, the buffer that differs ("-": none; several joined by +), what of it: a type, or dimensions joined by x
int main(int argc, char** argv) {
    for (int i = 1; i + 2 < argc; i += 3) {
        const std::string target = argv[i], name = argv[i + 1], what = argv[i + 2];
        Buffers b = good();
        std::vector<int64_t> section = {20, 12};
        if (name != "-") {
            if (what[0] >= '0' && what[0] <= '9') {
                std::vector<int64_t> dims;
                std::stringstream s(what);
                for (std::string n; std::getline(s, n, 'x');) {
                    dims.push_back(std::stoll(n));
                }
                std::stringstream names(name);
                for (std::string n; std::getline(names, n, '+');) {
                    (n == "section" ? section : b.at(n).dims) = dims;
                }
            } else {
                b.at(name).type = type_of(what);
            }
        }
        g_seen.clear();
        const ffi::Error e = call(target, b, section);
        if (e.code == ffi::ErrorCode::kOk) {
            printf("called%s\n", g_seen.c_str());
        } else {
            printf("refused %s%s\n", e.message.c_str(), g_seen.empty() ? "" : " AFTER THE CALL");
        }
    }
    return 0;
}
