// The XLA FFI targets: thin wrappers that unpack the call frame and forward to the plain C entry points.
// `MkSample` is cck_mk_sample; `CckRotary`, `CckCacheAppend` and `CckCacheAttention` are the sequence operators. Compiled only when CCK_FFI is defined and the XLA FFI headers
// are on the include path (they ship with jax; this repository does not carry them).
//
// Same binding as the reference's handler (src/diffusion/host.cuh:505-549): the platform stream,
// 1 + 74 untyped argument buffers (ext first), two results (positions, workspace) and the int32
// attributes samples, nsteps, flags; command-buffer compatible because nothing synchronises.
#ifdef CCK_FFI
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <string>

#include "../../include/cck_b200.h"
#include "xla/ffi/api/ffi.h"

namespace ffi = xla::ffi;

static ffi::Error mk_sample_ffi(cudaStream_t stream, ffi::RemainingArgs args, ffi::Result<ffi::AnyBuffer> out,
                                ffi::Result<ffi::AnyBuffer> ws, int32_t samples, int32_t nsteps, int32_t flags) {
    if (args.size() != CCK_NUM_INPUTS + 1) {
        return ffi::Error(ffi::ErrorCode::kInvalidArgument, "MkSample: wrong number of inputs");
    }
    auto ext = args.get<ffi::AnyBuffer>(0);
    if (ext.has_error()) {
        return ext.error();
    }
    const void* in[CCK_NUM_INPUTS];
    size_t bytes[CCK_NUM_INPUTS];
    for (int i = 0; i < CCK_NUM_INPUTS; i++) {
        auto buf = args.get<ffi::AnyBuffer>(i + 1);
        if (buf.has_error()) {
            return buf.error();
        }
        in[i] = buf->untyped_data();
        bytes[i] = buf->size_bytes();
    }
    const int rc = cck_mk_sample(stream, static_cast<const int*>(ext->untyped_data()), in, bytes, CCK_NUM_INPUTS,
                                 static_cast<float*>(out->untyped_data()), int(out->dimensions()[1]),
                                 ws->untyped_data(), ws->size_bytes(), samples, nsteps, flags);
    if (rc == CCK_OK) {
        return ffi::Error::Success();
    }
    return ffi::Error(rc == CCK_E_LAUNCH || rc == CCK_E_DEVICE ? ffi::ErrorCode::kInternal : ffi::ErrorCode::kInvalidArgument,
                      cck_last_error());
}

XLA_FFI_DEFINE_HANDLER_SYMBOL(MkSample, mk_sample_ffi,
                              ffi::Ffi::Bind()
                                  .Ctx<ffi::PlatformStream<cudaStream_t>>()
                                  .RemainingArgs()
                                  .Ret<ffi::AnyBuffer>()
                                  .Ret<ffi::AnyBuffer>()
                                  .Attr<int32_t>("samples")
                                  .Attr<int32_t>("nsteps")
                                  .Attr<int32_t>("flags"),
                              {ffi::Traits::kCmdBufferCompatible});

// ---- the sequence operators: descriptors from the buffers' shapes
static ffi::Error answer(int rc) {
    if (rc == CCK_OK) {
        return ffi::Error::Success();
    }
    return ffi::Error(rc == CCK_E_LAUNCH || rc == CCK_E_DEVICE ? ffi::ErrorCode::kInternal : ffi::ErrorCode::kInvalidArgument, cck_last_error());
}
static ffi::Error invalid(const char* target, const char* what) {
    return ffi::Error(ffi::ErrorCode::kInvalidArgument, std::string(target) + ": " + what);
}
// The C entry points take addresses and sizes: what a buffer holds is checked here, its type and every dimension.
static bool holds(ffi::AnyBuffer b, ffi::DataType type, std::initializer_list<int64_t> dims) {
    const auto d = b.dimensions();
    return b.element_type() == type && d.size() == dims.size() && std::equal(dims.begin(), dims.end(), d.begin());
}
static bool same_dims(ffi::AnyBuffer a, ffi::AnyBuffer b) {
    const auto d = a.dimensions(), e = b.dimensions();
    return d.size() == e.size() && std::equal(d.begin(), d.end(), e.begin());
}
static int64_t dim_of(ffi::AnyBuffer b, size_t i) {
    return i < b.dimensions().size() ? b.dimensions()[i] : 0;
}
// a size that the C entry points take in 32 bits; one that does not fit becomes one that they refuse
static int32_t size32(int64_t n) {
    return n >= 0 && n <= INT32_MAX ? int32_t(n) : -1;
}
// a dense tensor [rows][heads][dim]; a shape or type that is none gives one that the C entry point refuses
static cck_rows rows_of(ffi::AnyBuffer b) {
    const auto d = b.dimensions();
    cck_rows r{};
    r.data = b.untyped_data(), r.dtype = -1;
    if (d.size() == 3) {
        r.heads = size32(d[1]), r.head_stride = d[2], r.row_stride = d[1] * d[2];
        r.dtype = b.element_type() == ffi::DataType::BF16 ? CCK_BF16 : b.element_type() == ffi::DataType::F16 ? CCK_F16 : b.element_type() == ffi::DataType::F32 ? CCK_F32 : -1;
    }
    return r;
}
// each of these fills a descriptor, or says what does not fit
static const char* rotation_of(cck_rotation& r, ffi::AnyBuffer freq, ffi::AnyBuffer pos, int64_t rows, ffi::Span<const int64_t> section, int32_t adjacent) {
    const int64_t axes = int64_t(section.size()), pairs = dim_of(freq, 0);
    if (!holds(freq, ffi::DataType::F32, {pairs})) {
        return "freq is not f32 [pairs]";
    }
    if (!holds(pos, ffi::DataType::S32, {axes, rows}) && !(axes == 1 && holds(pos, ffi::DataType::S32, {rows}))) {
        return "pos is not s32 [axes][rows]";
    }
    r = cck_rotation{};
    r.axes = size32(axes), r.adjacent = adjacent, r.dims = size32(2 * pairs);
    for (int64_t a = 0; a < axes && a < 4; a++) {
        r.section[a] = size32(section[a]);
    }
    r.freq = static_cast<const float*>(freq.untyped_data()), r.pos = static_cast<const int32_t*>(pos.untyped_data());
    r.pos_stride = rows;
    return nullptr;
}
// scales are [pages][heads]; the head's dimensions follow from the codes' bytes, whose own shape is the caller's
static const char* cache_of(cck_cache& c, ffi::AnyBuffer k, ffi::AnyBuffer v, ffi::AnyBuffer k_scale, ffi::AnyBuffer v_scale, int32_t page_tokens) {
    const int64_t pages = dim_of(k_scale, 0), heads = dim_of(k_scale, 1);
    if (!holds(k_scale, ffi::DataType::F32, {pages, heads}) || !holds(v_scale, ffi::DataType::F32, {pages, heads})) {
        return "the cache's scales are not f32 [pages][heads]";
    }
    const int64_t tokens = page_tokens > 0 ? pages * heads * page_tokens : 0, bytes = int64_t(k.size_bytes());
    if (k.size_bytes() != k.element_count() || v.size_bytes() != v.element_count() || v.size_bytes() != k.size_bytes() || tokens == 0 || bytes % tokens != 0) {
        return "the cache's codes are not 8 bits for each page, head, token and dimension";
    }
    c = cck_cache{};
    c.k = k.untyped_data(), c.v = v.untyped_data();
    c.k_scale = static_cast<float*>(k_scale.untyped_data()), c.v_scale = static_cast<float*>(v_scale.untyped_data());
    c.page_tokens = page_tokens, c.pages = size32(pages), c.heads = size32(heads), c.dim = size32(bytes / tokens);
    return nullptr;
}
static const char* batch_of(cck_batch& b, ffi::AnyBuffer first, ffi::AnyBuffer len, ffi::AnyBuffer table, int64_t rows, int32_t max_new, int32_t max_len) {
    const int64_t sequences = dim_of(len, 0), columns = dim_of(table, 1);
    if (!holds(first, ffi::DataType::S32, {sequences + 1}) || !holds(len, ffi::DataType::S32, {sequences}) || !holds(table, ffi::DataType::S32, {sequences, columns})) {
        return "first, len and table are not s32 [sequences + 1], [sequences] and [sequences][pages]";
    }
    b = cck_batch{};
    b.sequences = size32(sequences), b.rows = size32(rows), b.max_new = max_new, b.max_len = max_len;
    b.table_pages = size32(columns), b.table_stride = columns;
    b.first = static_cast<const int32_t*>(first.untyped_data()), b.len = static_cast<const int32_t*>(len.untyped_data());
    b.table = static_cast<const int32_t*>(table.untyped_data());
    return nullptr;
}

// y = R(pos) x; x may be donated to y
static ffi::Error rotary_ffi(cudaStream_t stream, ffi::AnyBuffer x, ffi::AnyBuffer freq, ffi::AnyBuffer pos, ffi::Result<ffi::AnyBuffer> y, ffi::Span<const int64_t> section,
                             int32_t adjacent, int32_t inverse) {
    cck_rotation r;
    if (const char* what = rotation_of(r, freq, pos, dim_of(x, 0), section, adjacent)) {
        return invalid("CckRotary", what);
    }
    if (!same_dims(x, *y)) {
        return invalid("CckRotary", "x and y differ in shape");
    }
    const cck_rows from = rows_of(x), to = rows_of(*y);
    return answer(cck_rotary(stream, &r, size32(dim_of(x, 0)), size32(dim_of(x, 2)), &from, &to, inverse));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(CckRotary, rotary_ffi,
                              ffi::Ffi::Bind()
                                  .Ctx<ffi::PlatformStream<cudaStream_t>>()
                                  .Arg<ffi::AnyBuffer>()  // x
                                  .Arg<ffi::AnyBuffer>()  // freq
                                  .Arg<ffi::AnyBuffer>()  // pos
                                  .Ret<ffi::AnyBuffer>()  // y
                                  .Attr<ffi::Span<const int64_t>>("section")
                                  .Attr<int32_t>("adjacent")
                                  .Attr<int32_t>("inverse"),
                              {ffi::Traits::kCmdBufferCompatible});

// The cache's four buffers are results too, which the caller aliases to the operands (input_output_aliases): it is written in place
static ffi::Error cache_append_ffi(cudaStream_t stream, ffi::AnyBuffer kc, ffi::AnyBuffer vc, ffi::AnyBuffer ks, ffi::AnyBuffer vs, ffi::AnyBuffer k, ffi::AnyBuffer v,
                                   ffi::AnyBuffer q, ffi::AnyBuffer freq, ffi::AnyBuffer pos, ffi::AnyBuffer first, ffi::AnyBuffer len, ffi::AnyBuffer table,
                                   ffi::Result<ffi::AnyBuffer> kc_out, ffi::Result<ffi::AnyBuffer> vc_out, ffi::Result<ffi::AnyBuffer> ks_out,
                                   ffi::Result<ffi::AnyBuffer> vs_out, ffi::Result<ffi::AnyBuffer> q_out, ffi::Span<const int64_t> section, int32_t adjacent,
                                   int32_t page_tokens, int32_t max_new, int32_t max_len) {
    if (kc_out->untyped_data() != kc.untyped_data() || vc_out->untyped_data() != vc.untyped_data() || ks_out->untyped_data() != ks.untyped_data() ||
        vs_out->untyped_data() != vs.untyped_data()) {
        return invalid("CckCacheAppend", "the cache's results have to be aliased to its operands");
    }
    if (!same_dims(kc, *kc_out) || !same_dims(vc, *vc_out) || !same_dims(ks, *ks_out) || !same_dims(vs, *vs_out)) {
        return invalid("CckCacheAppend", "the cache's results differ from its operands in shape");
    }
    const int64_t rows = dim_of(k, 0);
    cck_rotation r;
    cck_cache c;
    cck_batch b;
    const char* what;
    if ((what = rotation_of(r, freq, pos, rows, section, adjacent)) || (what = cache_of(c, kc, vc, ks, vs, page_tokens)) ||
        (what = batch_of(b, first, len, table, rows, max_new, max_len))) {
        return invalid("CckCacheAppend", what);
    }
    if (!same_dims(k, v) || dim_of(q, 0) != rows || !same_dims(q, *q_out)) {
        return invalid("CckCacheAppend", "k and v, or q and the result, differ in shape, or k and q in rows");
    }
    if (dim_of(k, 2) != c.dim || dim_of(q, 2) != c.dim) {
        return invalid("CckCacheAppend", "heads of k, v and q have the cache's dimensions");
    }
    const cck_rows kr = rows_of(k), vr = rows_of(v), from = rows_of(q), to = rows_of(*q_out);
    return answer(cck_cache_append(stream, &c, &b, &kr, &vr, &r, &from, &to, nullptr));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(CckCacheAppend, cache_append_ffi,
                              ffi::Ffi::Bind()
                                  .Ctx<ffi::PlatformStream<cudaStream_t>>()
                                  .Arg<ffi::AnyBuffer>()  // codes of the keys
                                  .Arg<ffi::AnyBuffer>()  // codes of the values
                                  .Arg<ffi::AnyBuffer>()  // scales of the keys
                                  .Arg<ffi::AnyBuffer>()  // scales of the values
                                  .Arg<ffi::AnyBuffer>()  // k
                                  .Arg<ffi::AnyBuffer>()  // v
                                  .Arg<ffi::AnyBuffer>()  // q
                                  .Arg<ffi::AnyBuffer>()  // freq
                                  .Arg<ffi::AnyBuffer>()  // pos
                                  .Arg<ffi::AnyBuffer>()  // first
                                  .Arg<ffi::AnyBuffer>()  // len
                                  .Arg<ffi::AnyBuffer>()  // table
                                  .Ret<ffi::AnyBuffer>()
                                  .Ret<ffi::AnyBuffer>()
                                  .Ret<ffi::AnyBuffer>()
                                  .Ret<ffi::AnyBuffer>()
                                  .Ret<ffi::AnyBuffer>()  // q rotated
                                  .Attr<ffi::Span<const int64_t>>("section")
                                  .Attr<int32_t>("adjacent")
                                  .Attr<int32_t>("page_tokens")
                                  .Attr<int32_t>("max_new")
                                  .Attr<int32_t>("max_len"),
                              {ffi::Traits::kCmdBufferCompatible});

static ffi::Error cache_attention_ffi(cudaStream_t stream, ffi::AnyBuffer kc, ffi::AnyBuffer vc, ffi::AnyBuffer ks, ffi::AnyBuffer vs, ffi::AnyBuffer q, ffi::AnyBuffer first,
                                      ffi::AnyBuffer len, ffi::AnyBuffer table, ffi::Result<ffi::AnyBuffer> out, ffi::Result<ffi::AnyBuffer> lse,
                                      ffi::Result<ffi::AnyBuffer> ws, float softmax_scale, int32_t causal, int32_t window, int32_t page_tokens, int32_t max_new,
                                      int32_t max_len) {
    cck_cache c;
    cck_batch b;
    const char* what;
    if ((what = cache_of(c, kc, vc, ks, vs, page_tokens)) || (what = batch_of(b, first, len, table, dim_of(q, 0), max_new, max_len))) {
        return invalid("CckCacheAttention", what);
    }
    if (dim_of(q, 2) != c.dim || !same_dims(q, *out)) {
        return invalid("CckCacheAttention", "q and out differ in shape, or heads have not the cache's dimensions");
    }
    if (!holds(*lse, ffi::DataType::F32, {dim_of(q, 0), dim_of(q, 1)})) {
        return invalid("CckCacheAttention", "lse is not f32 [rows][heads]");
    }
    const cck_rows from = rows_of(q), to = rows_of(*out);
    return answer(cck_cache_attention(stream, &c, &b, &from, &to, static_cast<float*>(lse->untyped_data()), softmax_scale, causal, window, ws->untyped_data(),
                                      ws->size_bytes()));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(CckCacheAttention, cache_attention_ffi,
                              ffi::Ffi::Bind()
                                  .Ctx<ffi::PlatformStream<cudaStream_t>>()
                                  .Arg<ffi::AnyBuffer>()  // codes of the keys
                                  .Arg<ffi::AnyBuffer>()  // codes of the values
                                  .Arg<ffi::AnyBuffer>()  // scales of the keys
                                  .Arg<ffi::AnyBuffer>()  // scales of the values
                                  .Arg<ffi::AnyBuffer>()  // q
                                  .Arg<ffi::AnyBuffer>()  // first
                                  .Arg<ffi::AnyBuffer>()  // len
                                  .Arg<ffi::AnyBuffer>()  // table
                                  .Ret<ffi::AnyBuffer>()  // out
                                  .Ret<ffi::AnyBuffer>()  // lse
                                  .Ret<ffi::AnyBuffer>()  // workspace
                                  .Attr<float>("softmax_scale")
                                  .Attr<int32_t>("causal")
                                  .Attr<int32_t>("window")
                                  .Attr<int32_t>("page_tokens")
                                  .Attr<int32_t>("max_new")
                                  .Attr<int32_t>("max_len"),
                              {ffi::Traits::kCmdBufferCompatible});
#endif
