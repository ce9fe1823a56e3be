// The XLA FFI targets: thin wrappers that unpack the call frame and forward to the plain C entry points.
// `MkSample` is cck_mk_sample; `CckRotary`, `CckCacheAppend` and `CckCacheAttention` are the sequence operators. Compiled only when CCK_FFI is defined and the XLA FFI headers
// are on the include path (they ship with jax; this repository does not carry them).
//
// Same binding as the reference's handler (src/diffusion/host.cuh:505-549): the platform stream,
// 1 + 74 untyped argument buffers (ext first), two results (positions, workspace) and the int32
// attributes samples, nsteps, flags; command-buffer compatible because nothing synchronises.
#ifdef CCK_FFI
#include <cuda_runtime.h>

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
// a dense tensor [rows][heads][dim]; a shape or type that is none gives one that the C entry point refuses
static cck_rows rows_of(ffi::AnyBuffer b) {
    const auto d = b.dimensions();
    cck_rows r{};
    r.data = b.untyped_data(), r.dtype = -1;
    if (d.size() == 3) {
        r.heads = int32_t(d[1]), r.head_stride = d[2], r.row_stride = d[1] * d[2];
        r.dtype = b.element_type() == ffi::DataType::BF16 ? CCK_BF16 : b.element_type() == ffi::DataType::F16 ? CCK_F16 : b.element_type() == ffi::DataType::F32 ? CCK_F32 : -1;
    }
    return r;
}
static cck_rotation rotation_of(ffi::AnyBuffer freq, ffi::AnyBuffer pos, ffi::Span<const int64_t> section, int32_t adjacent) {
    cck_rotation r{};
    r.axes = int32_t(section.size()), r.adjacent = adjacent, r.dims = int32_t(2 * freq.element_count());
    for (size_t a = 0; a < section.size() && a < 4; a++) {
        r.section[a] = int32_t(section[a]);
    }
    r.freq = static_cast<const float*>(freq.untyped_data()), r.pos = static_cast<const int32_t*>(pos.untyped_data());
    r.pos_stride = section.size() ? int64_t(pos.element_count() / section.size()) : 0;
    return r;
}
// k_scale is [pages][heads]; the head's dimensions follow from the codes' bytes
static cck_cache cache_of(ffi::AnyBuffer k, ffi::AnyBuffer v, ffi::AnyBuffer k_scale, ffi::AnyBuffer v_scale, int32_t page_tokens) {
    const auto d = k_scale.dimensions();
    cck_cache c{};
    c.k = k.untyped_data(), c.v = v.untyped_data();
    c.k_scale = static_cast<float*>(k_scale.untyped_data()), c.v_scale = static_cast<float*>(v_scale.untyped_data());
    c.page_tokens = page_tokens;
    if (d.size() == 2 && v_scale.element_count() == k_scale.element_count() && v.size_bytes() == k.size_bytes()) {
        c.pages = int32_t(d[0]), c.heads = int32_t(d[1]);
        const int64_t tokens = d[0] * d[1] * page_tokens;
        c.dim = tokens > 0 && int64_t(k.size_bytes()) % tokens == 0 ? int32_t(int64_t(k.size_bytes()) / tokens) : 0;
    }
    return c;
}
static cck_batch batch_of(ffi::AnyBuffer first, ffi::AnyBuffer len, ffi::AnyBuffer table, int64_t rows, int32_t max_new, int32_t max_len) {
    const auto d = table.dimensions();
    cck_batch b{};
    b.sequences = int32_t(len.element_count()), b.rows = int32_t(rows), b.max_new = max_new, b.max_len = max_len;
    if (d.size() == 2 && d[0] == int64_t(len.element_count()) && first.element_count() == len.element_count() + 1) {
        b.table_pages = int32_t(d[1]), b.table_stride = d[1];
    }
    b.first = static_cast<const int32_t*>(first.untyped_data()), b.len = static_cast<const int32_t*>(len.untyped_data());
    b.table = static_cast<const int32_t*>(table.untyped_data());
    return b;
}
static int64_t dim_of(ffi::AnyBuffer b, size_t i) {
    return i < b.dimensions().size() ? b.dimensions()[i] : 0;
}

// y = R(pos) x; x may be donated to y
static ffi::Error rotary_ffi(cudaStream_t stream, ffi::AnyBuffer x, ffi::AnyBuffer freq, ffi::AnyBuffer pos, ffi::Result<ffi::AnyBuffer> y, ffi::Span<const int64_t> section,
                             int32_t adjacent, int32_t inverse) {
    const cck_rotation r = rotation_of(freq, pos, section, adjacent);
    if (r.pos_stride != dim_of(x, 0) || y->element_count() != x.element_count()) {
        return ffi::Error(ffi::ErrorCode::kInvalidArgument, "CckRotary: positions or result do not fit the rows");
    }
    const cck_rows from = rows_of(x), to = rows_of(*y);
    return answer(cck_rotary(stream, &r, int(dim_of(x, 0)), int(dim_of(x, 2)), &from, &to, inverse));
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
        return ffi::Error(ffi::ErrorCode::kInvalidArgument, "CckCacheAppend: the cache's results have to be aliased to its operands");
    }
    const cck_rotation r = rotation_of(freq, pos, section, adjacent);
    const int64_t rows = dim_of(k, 0);
    if (r.pos_stride != rows || dim_of(v, 0) != rows || dim_of(q, 0) != rows || q_out->element_count() != q.element_count()) {
        return ffi::Error(ffi::ErrorCode::kInvalidArgument, "CckCacheAppend: k, v, q, their positions and the result differ in rows");
    }
    const cck_cache c = cache_of(kc, vc, ks, vs, page_tokens);
    if (dim_of(k, 2) != c.dim || dim_of(v, 2) != c.dim || dim_of(q, 2) != c.dim) {
        return ffi::Error(ffi::ErrorCode::kInvalidArgument, "CckCacheAppend: heads of k, v and q have the cache's dimensions");
    }
    const cck_batch b = batch_of(first, len, table, rows, max_new, max_len);
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
    const cck_cache c = cache_of(kc, vc, ks, vs, page_tokens);
    const cck_batch b = batch_of(first, len, table, dim_of(q, 0), max_new, max_len);
    if (dim_of(q, 2) != c.dim || out->element_count() != q.element_count() || int64_t(lse->element_count()) != dim_of(q, 0) * dim_of(q, 1)) {
        return ffi::Error(ffi::ErrorCode::kInvalidArgument, "CckCacheAttention: q, out and lse do not fit each other or the cache");
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
