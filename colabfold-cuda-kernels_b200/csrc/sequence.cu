// The sequence operators' C entry points: checks of the arguments, the choice of a kernel, the launch.
// Declarations: include/cck_b200.h.
#include <atomic>
#include <cstdio>

#include "cache_append.cuh"
#include "cache_attention_tile.cuh"
#include "report.h"

using namespace cck;
using namespace cck::seq;

namespace {

constexpr int kMaxDevices = 64;

int refuse(int code, const char* op, const char* what) {
    char text[256];
    snprintf(text, sizeof text, "%s: %s", op, what);
    return report(code, text);
}
int launched(const char* op, cudaError_t err) {
    return err == cudaSuccess ? CCK_OK : refuse(CCK_E_LAUNCH, op, cudaGetErrorString(err));
}

// the current device's multiprocessors; `data` has to be its memory
int device_of(const char* op, const void* data, int& sms) {
    static std::atomic<int> known[kMaxDevices];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
        cudaGetLastError();
        return refuse(CCK_E_DEVICE, op, "no CUDA device");
    }
    sms = known[dev].load(std::memory_order_relaxed);
    if (sms == 0) {
        int major = 0, count = 0;
        if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
            cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || major != 10) {
            cudaGetLastError();
            return refuse(CCK_E_DEVICE, op, "this library holds sm_100a code only");
        }
        known[dev].store(sms = count, std::memory_order_relaxed);
    }
    cudaPointerAttributes at;
    if (cudaPointerGetAttributes(&at, data) != cudaSuccess || at.type == cudaMemoryTypeUnregistered) {
        cudaGetLastError();
        return refuse(CCK_E_DEVICE, op, "a tensor is not in device memory");
    }
    if (at.type == cudaMemoryTypeDevice && at.device != dev) {
        return refuse(CCK_E_DEVICE, op, "a tensor is on another device than the current one");
    }
    return CCK_OK;
}

int size_of(int dtype) {
    return dtype == CCK_F32 ? 4 : 2;
}
bool aligned(const void* p, size_t n) {
    return reinterpret_cast<uintptr_t>(p) % n == 0;
}
// what is wrong with a tensor: null, or the text of the refusal; `bytes`: what data and strides are multiples of
int check_rows(const char* op, const cck_rows* x, const char* name, int bytes, bool f32) {
    char text[128];
    auto say = [&](const char* what) {
        snprintf(text, sizeof text, "%s %s", name, what);
        return text;
    };
    if (!x || !x->data) {
        return refuse(CCK_E_SHAPE, op, say("is null"));
    }
    if (x->dtype != CCK_BF16 && x->dtype != CCK_F16 && !(f32 && x->dtype == CCK_F32)) {
        return refuse(CCK_E_FLAGS, op, say("has a type that is not built"));
    }
    if (x->heads < 1 || x->row_stride < 0 || x->head_stride < 0) {
        return refuse(CCK_E_SHAPE, op, say("has no heads, or a negative stride"));
    }
    if (!aligned(x->data, bytes ? bytes : size_of(x->dtype)) || (bytes && (x->row_stride * size_of(x->dtype) % bytes || x->head_stride * size_of(x->dtype) % bytes))) {
        return refuse(CCK_E_SHAPE, op, say("is not aligned"));
    }
    return CCK_OK;
}
int check_rotation(const char* op, const cck_rotation* r, int dim) {
    if (r->dims < 0 || r->dims % 2 || r->dims > dim || r->axes < 1 || r->axes > 4) {
        return refuse(CCK_E_SHAPE, op, "rotation: dims is even and at most a head's, axes 1 to 4");
    }
    int64_t pairs = 0;
    for (int a = 0; a < r->axes; a++) {
        if (r->section[a] < 0) {
            return refuse(CCK_E_SHAPE, op, "rotation: a section is negative");
        }
        pairs += r->section[a];
    }
    if (pairs != r->dims / 2) {
        return refuse(CCK_E_SHAPE, op, "rotation: the sections do not add up to dims / 2");
    }
    if (r->dims && (!r->freq || !r->pos || !aligned(r->freq, 4) || !aligned(r->pos, 4))) {
        return refuse(CCK_E_SHAPE, op, "rotation: freq or pos is null or not aligned");
    }
    return CCK_OK;
}
int check_cache(const char* op, const cck_cache* c) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) {
        return refuse(CCK_E_SHAPE, op, "the cache or a part of it is null");
    }
    if (c->pages < 1 || c->heads < 1) {
        return refuse(CCK_E_SHAPE, op, "the cache has no pages or no heads");
    }
    if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128) {
        return refuse(CCK_E_SHAPE, op, "a page holds 16, 32, 64 or 128 tokens");
    }
    if (c->dim != 32 && c->dim != 64 && c->dim != 96 && c->dim != 128) {
        return refuse(CCK_E_SHAPE, op, "the cache's heads have 32, 64, 96 or 128 dimensions");
    }
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4)) {
        return refuse(CCK_E_SHAPE, op, "the cache is not aligned");
    }
    return CCK_OK;
}
int check_batch(const char* op, const cck_batch* b) {
    if (!b || !b->first || !b->len || !b->table || !aligned(b->first, 4) || !aligned(b->len, 4) || !aligned(b->table, 4)) {
        return refuse(CCK_E_SHAPE, op, "the batch or an array of it is null or not aligned");
    }
    if (b->sequences < 0 || b->rows < 0 || b->max_new < 0 || b->max_len < 0 || b->table_pages < 1 || b->table_stride < 0) {
        return refuse(CCK_E_SHAPE, op, "a size of the batch is negative, or its table has no pages");
    }
    return CCK_OK;
}

// an input and its output: the same type and heads, and no element of the output twice
int check_pair(const char* op, const cck_rows* x, const cck_rows* out, int64_t rows, int dim) {
    if (x->dtype != out->dtype || x->heads != out->heads) {
        return refuse(CCK_E_SHAPE, op, "input and output differ in type or heads");
    }
    if (x->data == out->data && (x->row_stride != out->row_stride || x->head_stride != out->head_stride)) {
        return refuse(CCK_E_SHAPE, op, "in place, input and output have the same strides");
    }
    int64_t n = rows, m = out->heads, ns = out->row_stride, ms = out->head_stride;
    if (n <= 1 || (m > 1 && ns > ms)) { // n: the dimension with the smaller stride
        const int64_t t = n, ts = ns;
        n = m, ns = ms, m = t, ms = ts;
    }
    const int64_t inner = n > 1 ? (n - 1) * ns + dim : dim;
    if ((n > 1 && ns < dim) || (m > 1 && ms < inner)) {
        return refuse(CCK_E_SHAPE, op, "elements of the output overlap");
    }
    return CCK_OK;
}

// A head's pairs a thread takes at once: the most, up to 16 bytes, that the sizes and the alignment of both tensors allow
int rotary_vector(const cck_rotation& r, int dim, const cck_rows& x, const cck_rows& y) {
    const int size = size_of(x.dtype);
    for (int v = 16 / size; v > 1; v /= 2) {
        const int64_t strides = x.row_stride | x.head_stride | y.row_stride | y.head_stride;
        if (r.dims / 2 % v == 0 && (dim - r.dims) % v == 0 && strides % v == 0 && aligned(x.data, v * size) && aligned(y.data, v * size)) {
            return v;
        }
    }
    return 1;
}
RotaryShape rotary_shape(const cck_rotation& r, int rows, int dim, const cck_rows& x, const cck_rows& y, bool inverse, int v, int sms) {
    RotaryShape s{};
    s.rows = rows, s.dim = dim, s.heads = x.heads, s.sign = inverse ? -1 : 1;
    s.x = x.data, s.y = y.data, s.xr = x.row_stride, s.xh = x.head_stride, s.yr = y.row_stride, s.yh = y.head_stride;
    s.rot_items = r.dims / 2 / v;
    s.items = s.rot_items + (x.data == y.data ? 0 : ceil_div(dim - r.dims, 2 * v));
    // threads that share a row's heads: few, since each computes the row's angles anew, but enough to fill the GPU
    const int64_t want = int64_t(sms) * 2048, one = int64_t(rows) * (s.items ? s.items : 1);
    s.hs = int(one >= want ? 1 : (want + one - 1) / one);
    s.hs = s.hs < x.heads ? s.hs : x.heads;
    return s;
}
int64_t rotary_blocks(const RotaryShape& s, int threads) {
    const int slots = threads / s.items;
    return (int64_t(s.rows) * s.hs + slots - 1) / slots;
}

template <class T>
cudaError_t launch_rotary(cudaStream_t st, const cck_rotation& r, const RotaryShape& s, int v, int64_t blocks, int threads) {
    auto go = [&](auto kernel) {
        kernel<<<unsigned(blocks), threads, 0, st>>>(r, s);
        return cudaGetLastError();
    };
    constexpr int kMost = 16 / sizeof(T);
    switch (v) {
    case 8: return go(rotary_kernel<T, kMost>);
    case 4: return go(rotary_kernel<T, 4>);
    case 2: return go(rotary_kernel<T, 2>);
    default: return go(rotary_kernel<T, 1>);
    }
}

template <class T>
cudaError_t launch_append(cudaStream_t st, const AppendArgs& a, int v, unsigned blocks, size_t smem) {
    auto go = [&](auto kernel) {
        if (smem > 48 * 1024) {
            if (cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem))) {
                return e;
            }
        }
        kernel<<<blocks, kAppendThreads, smem, st>>>(a);
        return cudaGetLastError();
    };
    constexpr int kMost = 16 / sizeof(T);
    switch (v) {
    case 8: return go(append_kernel<T, kMost>);
    case 4: return go(append_kernel<T, 4>);
    case 2: return go(append_kernel<T, 2>);
    default: return go(append_kernel<T, 1>);
    }
}

// How an attention call is cut up: whole units, a block each, or equal shares of the line of all units
struct Plan {
    int nt;                 // tiles of 8 rows of a warp of decode_kernel; 0: tile_kernel
    int granule, tile_rows; // keys and rows of a step
    int row_tiles;          // of a sequence
    int64_t blocks;
    bool shares;
    int merge_y;
    size_t part_bytes, ml_bytes, bytes; // of the workspace
};
Plan make_plan(const cck_cache& c, const cck_batch& b, int q_heads, int sms) {
    Plan p{};
    const int64_t rows = int64_t(b.max_new) * (q_heads / c.heads);
    p.nt = rows <= 8 ? 1 : rows <= 16 ? 2 : 0;
    p.granule = p.nt ? granule_of(c.dim) : kTileKeys, p.tile_rows = p.nt ? 8 * p.nt : kUnitRows;
    p.row_tiles = int((rows + p.tile_rows - 1) / p.tile_rows);
    const int64_t units = int64_t(b.sequences) * c.heads * p.row_tiles, slots = (p.nt == 0 ? 1 : p.nt == 1 ? 3 : 2) * sms;
    const int64_t granules = int64_t(b.max_len) / p.granule + 2;
    const int least = p.nt ? 2 * kDecodeWarps : 2; // granules of a share
    p.shares = granules > 2 * least && units < 8 * slots;
    const int64_t most = (units * granules + least - 1) / least;
    p.blocks = !p.shares ? units : most < slots ? most : slots;
    if (p.shares) {
        p.merge_y = p.nt == 0 ? 16 : units < 64 ? p.tile_rows : 1;
        p.part_bytes = size_t(2 * p.blocks) * p.tile_rows * c.dim * 4;
        p.ml_bytes = size_t(2 * p.blocks) * p.tile_rows * 8;
        p.bytes = p.part_bytes + p.ml_bytes + size_t(p.blocks) * sizeof(Split);
    }
    return p;
}
// the attribute that a kernel of more than 48 KB needs, once a device
template <class K>
cudaError_t allow_shared(K kernel, int bytes, std::atomic<bool>* ready) {
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) {
        return e;
    }
    if (!ready[dev].load(std::memory_order_relaxed)) {
        if (cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) {
            return e;
        }
        ready[dev].store(true, std::memory_order_relaxed);
    }
    return cudaSuccess;
}
template <class T, int D, int NT>
cudaError_t launch_decode(cudaStream_t st, const AttentionArgs& a, unsigned blocks) {
    static std::atomic<bool> ready[kMaxDevices];
    if (cudaError_t e = allow_shared(decode_kernel<T, D, NT>, DecodeShape<D, NT>::kSmem, ready)) {
        return e;
    }
    decode_kernel<T, D, NT><<<blocks, kDecodeWarps * 32, DecodeShape<D, NT>::kSmem, st>>>(a);
    return cudaGetLastError();
}
template <class T, int D>
cudaError_t launch_tile(cudaStream_t st, const AttentionArgs& a, unsigned blocks) {
    static std::atomic<bool> ready[kMaxDevices];
    if (cudaError_t e = allow_shared(tile_kernel<T, D>, TileShape<T, D>::kSmem, ready)) {
        return e;
    }
    tile_kernel<T, D><<<blocks, kTileThreads, TileShape<T, D>::kSmem, st>>>(a);
    return cudaGetLastError();
}
template <class T, int D>
cudaError_t launch_attention(cudaStream_t st, const AttentionArgs& a, const Plan& p) {
    const unsigned blocks = unsigned(p.blocks);
    return p.nt == 0 ? launch_tile<T, D>(st, a, blocks) : p.nt == 1 ? launch_decode<T, D, 1>(st, a, blocks) : launch_decode<T, D, 2>(st, a, blocks);
}
template <class T>
cudaError_t launch_attention(cudaStream_t st, const AttentionArgs& a, const Plan& p) {
    const cudaError_t e = a.cache.dim == 32   ? launch_attention<T, 32>(st, a, p)
                          : a.cache.dim == 64 ? launch_attention<T, 64>(st, a, p)
                          : a.cache.dim == 96 ? launch_attention<T, 96>(st, a, p)
                                              : launch_attention<T, 128>(st, a, p);
    if (e || !p.shares) {
        return e;
    }
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute dependent;
    dependent.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    dependent.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(unsigned(p.blocks), unsigned(p.merge_y)), cfg.blockDim = dim3(kMergeWarps * 32), cfg.stream = st, cfg.attrs = &dependent, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, merge_kernel<T>, a);
}

} // namespace

extern "C" {

int cck_rotary(void* stream, const cck_rotation* rotation, int rows, int dim, const cck_rows* x, const cck_rows* y, int inverse) {
    const char* op = "cck_rotary";
    if (!rotation || rows < 0 || dim < 1 || dim > 1024) {
        return refuse(CCK_E_SHAPE, op, "rotation is null, rows is negative or dim is not 1 to 1024");
    }
    int e;
    if ((e = check_rotation(op, rotation, dim)) || (e = check_rows(op, x, "x", 0, true)) || (e = check_rows(op, y, "y", 0, true)) || (e = check_pair(op, x, y, rows, dim))) {
        return e;
    }
    int sms = 0;
    if ((e = device_of(op, x->data, sms)) || (e = device_of(op, y->data, sms))) {
        return e;
    }
    if (rows == 0) {
        return CCK_OK;
    }
    const int v = rotary_vector(*rotation, dim, *x, *y);
    const RotaryShape s = rotary_shape(*rotation, rows, dim, *x, *y, inverse != 0, v, sms);
    if (s.items == 0) { // in place and nothing turns
        return CCK_OK;
    }
    const int threads = s.items > 256 ? 512 : 256;
    const int64_t blocks = rotary_blocks(s, threads);
    if (blocks > 0x7fffffff) {
        return refuse(CCK_E_SHAPE, op, "too many rows for one launch");
    }
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (x->dtype) {
    case CCK_BF16: return launched(op, launch_rotary<__nv_bfloat16>(st, *rotation, s, v, blocks, threads));
    case CCK_F16: return launched(op, launch_rotary<__half>(st, *rotation, s, v, blocks, threads));
    default: return launched(op, launch_rotary<float>(st, *rotation, s, v, blocks, threads));
    }
}

int cck_cache_append(void* stream, const cck_cache* cache, const cck_batch* batch, const cck_rows* k, const cck_rows* v, const cck_rotation* rotation, const cck_rows* q,
                     const cck_rows* q_out, int32_t* status) {
    const char* op = "cck_cache_append";
    int e;
    if ((e = check_cache(op, cache)) || (e = check_batch(op, batch)) || (e = check_rows(op, k, "k", 16, true)) || (e = check_rows(op, v, "v", 16, true))) {
        return e;
    }
    if (k->dtype != v->dtype || k->heads != cache->heads || v->heads != cache->heads) {
        return refuse(CCK_E_SHAPE, op, "k and v have the cache's heads and one type");
    }
    if (rotation && (e = check_rotation(op, rotation, cache->dim))) {
        return e;
    }
    if (q) {
        if (!rotation) {
            return refuse(CCK_E_SHAPE, op, "queries are rotated, but there is no rotation");
        }
        if ((e = check_rows(op, q, "q", 0, true)) || (e = check_rows(op, q_out, "q_out", 0, true)) || (e = check_pair(op, q, q_out, batch->rows, cache->dim))) {
            return e;
        }
        if (q->dtype != k->dtype) {
            return refuse(CCK_E_SHAPE, op, "q has the type of k and v");
        }
    }
    if (status && !aligned(status, 4)) {
        return refuse(CCK_E_SHAPE, op, "status is not aligned");
    }
    int sms = 0;
    if ((e = device_of(op, cache->k, sms)) || (e = device_of(op, k->data, sms))) {
        return e;
    }
    AppendArgs a{};
    a.cache = *cache, a.batch = *batch, a.k = k->data, a.v = v->data, a.status = status;
    a.kr = k->row_stride, a.kh = k->head_stride, a.vr = v->row_stride, a.vh = v->head_stride;
    if (rotation) {
        a.rotation = *rotation;
    }
    const int P = cache->page_tokens;
    a.blocks_per_seq = batch->max_new ? (batch->max_new + P - 2) / P + 1 : 0;
    const int64_t kv = int64_t(batch->sequences) * a.blocks_per_seq * cache->heads;
    int64_t more = 0;
    int vec = 1;
    if (q && batch->rows) {
        vec = rotary_vector(*rotation, cache->dim, *q, *q_out);
        a.q = rotary_shape(*rotation, batch->rows, cache->dim, *q, *q_out, false, vec, sms);
        more = a.q.items ? rotary_blocks(a.q, kAppendThreads) : 0;
    }
    if (kv + more > 0x7fffffff) {
        return refuse(CCK_E_SHAPE, op, "too many rows for one launch");
    }
    if (kv + more == 0) {
        return CCK_OK;
    }
    a.kv_blocks = int(kv);
    const size_t smem = append_smem(batch->max_new < P ? batch->max_new : P, cache->dim, size_of(k->dtype));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (k->dtype) {
    case CCK_BF16: return launched(op, launch_append<__nv_bfloat16>(st, a, vec, unsigned(kv + more), smem));
    case CCK_F16: return launched(op, launch_append<__half>(st, a, vec, unsigned(kv + more), smem));
    default: return launched(op, launch_append<float>(st, a, vec, unsigned(kv + more), smem));
    }
}

size_t cck_cache_attention_workspace_bytes(const cck_cache* cache, const cck_batch* batch, int q_heads) {
    const char* op = "cck_cache_attention_workspace_bytes";
    int sms = 0;
    if (check_cache(op, cache) || check_batch(op, batch) || q_heads < 1 || q_heads % cache->heads || device_of(op, cache->k, sms)) {
        return 0;
    }
    return make_plan(*cache, *batch, q_heads, sms).bytes;
}

int cck_cache_attention(void* stream, const cck_cache* cache, const cck_batch* batch, const cck_rows* q, const cck_rows* out, float* lse, float softmax_scale, int causal,
                        int window, void* ws, size_t ws_bytes) {
    const char* op = "cck_cache_attention";
    int e;
    if ((e = check_cache(op, cache)) || (e = check_batch(op, batch)) || (e = check_rows(op, q, "q", 16, false)) || (e = check_rows(op, out, "out", 16, false)) ||
        (e = check_pair(op, q, out, batch->rows, cache->dim))) {
        return e;
    }
    if (q->heads % cache->heads) {
        return refuse(CCK_E_SHAPE, op, "the heads of q are no multiple of the cache's");
    }
    if (window < 0 || !(softmax_scale - softmax_scale == 0.f)) {
        return refuse(CCK_E_SHAPE, op, "window is negative or softmax_scale is not finite");
    }
    if (lse && !aligned(lse, 4)) {
        return refuse(CCK_E_SHAPE, op, "lse is not aligned");
    }
    int sms = 0;
    if ((e = device_of(op, cache->k, sms)) || (e = device_of(op, q->data, sms)) || (e = device_of(op, out->data, sms))) {
        return e;
    }
    if (batch->sequences == 0 || batch->rows == 0 || batch->max_new == 0) {
        return CCK_OK;
    }
    const Plan p = make_plan(*cache, *batch, q->heads, sms);
    if (ws_bytes < p.bytes || (p.bytes && (!ws || !aligned(ws, 16)))) {
        return refuse(CCK_E_WORKSPACE, op, "the workspace is too small, null or not aligned");
    }
    if (p.blocks > 0x7fffffff) {
        return refuse(CCK_E_SHAPE, op, "too many rows for one launch");
    }
    AttentionArgs a{};
    a.cache = *cache, a.batch = *batch, a.q = q->data, a.out = out->data, a.lse = lse;
    a.qr = q->row_stride, a.qh = q->head_stride, a.or_ = out->row_stride, a.oh = out->head_stride;
    a.scale_log2 = softmax_scale * 1.4426950408889634f;
    a.q_heads = q->heads, a.group = q->heads / cache->heads, a.causal = causal != 0, a.window = window;
    a.granule_shift = __builtin_ctz(p.granule), a.unit_cost = p.nt ? 8 : 3, a.page_shift = __builtin_ctz(cache->page_tokens);
    a.tile_rows = p.tile_rows, a.row_tiles = p.row_tiles;
    if (p.shares) {
        a.part_o = static_cast<float*>(ws), a.part_ml = reinterpret_cast<float*>(static_cast<char*>(ws) + p.part_bytes);
        a.splits = reinterpret_cast<Split*>(static_cast<char*>(ws) + p.part_bytes + p.ml_bytes);
    }
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return launched(op, q->dtype == CCK_BF16 ? launch_attention<__nv_bfloat16>(st, a, p) : launch_attention<__half>(st, a, p));
}

} // extern "C"
