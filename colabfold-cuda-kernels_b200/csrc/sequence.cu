// The sequence operators' C entry points: checks of the arguments, the choice of a kernel, the launch.
// Declarations: include/cck_b200.h.
#include <atomic>
#include <cstdio>
#include <initializer_list>
#include <type_traits>

#include "cache_append.cuh"
#include "cache_attention_tile.cuh"
#include "report.h"

using namespace cck;
using namespace cck::seq;

namespace {

constexpr int kMaxDevices = 64;
std::atomic<int> g_lose{-1}; // cck_set_lost_copy_test

int refuse(int code, const char* op, const char* what) {
    char text[256];
    snprintf(text, sizeof text, "%s: %s", op, what);
    return report(code, text);
}
int launched(const char* op, cudaError_t err) {
    return err == cudaSuccess ? CCK_OK : refuse(CCK_E_LAUNCH, op, cudaGetErrorString(err));
}

// the current device's multiprocessors; what `data` points to (null: nothing) has to be memory that it can read
int device_of(const char* op, std::initializer_list<const void*> data, int& sms) {
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
    for (const void* p : data) {
        cudaPointerAttributes at;
        if (p && (cudaPointerGetAttributes(&at, p) != cudaSuccess || at.type == cudaMemoryTypeUnregistered)) {
            cudaGetLastError();
            return refuse(CCK_E_DEVICE, op, "a tensor is not in device memory");
        }
        if (p && at.type == cudaMemoryTypeDevice && at.device != dev) {
            return refuse(CCK_E_DEVICE, op, "a tensor is on another device than the current one");
        }
    }
    return CCK_OK;
}

int size_of(int dtype) {
    return dtype == CCK_F32 ? 4 : 2;
}
bool aligned(const void* p, size_t n) {
    return reinterpret_cast<uintptr_t>(p) % n == 0;
}
// a tensor of `rows` rows; `bytes`: what data and strides are multiples of. One without rows may have no memory either
int check_rows(const char* op, const cck_rows* x, const char* name, int rows, int bytes, bool f32) {
    char text[128];
    auto say = [&](const char* what) {
        snprintf(text, sizeof text, "%s %s", name, what);
        return text;
    };
    if (!x || (!x->data && rows)) {
        return refuse(CCK_E_SHAPE, op, say("is null"));
    }
    if (x->dtype != CCK_BF16 && x->dtype != CCK_F16 && !(f32 && x->dtype == CCK_F32)) {
        return refuse(CCK_E_FLAGS, op, say("has a type that is not built"));
    }
    if (x->heads < 1 || x->heads > kMostHeads || x->row_stride < 0 || x->head_stride < 0) {
        return refuse(CCK_E_SHAPE, op, say("has no heads, more than 65536, or a negative stride"));
    }
    if (!aligned(x->data, bytes ? bytes : size_of(x->dtype)) || (bytes && (x->row_stride * size_of(x->dtype) % bytes || x->head_stride * size_of(x->dtype) % bytes))) {
        return refuse(CCK_E_SHAPE, op, say("is not aligned"));
    }
    return CCK_OK;
}
int check_rotation(const char* op, const cck_rotation* r, int rows, int dim) {
    if (r->dims < 0 || r->dims % 2 || r->dims > dim || r->axes < 1 || r->axes > 4) {
        return refuse(CCK_E_SHAPE, op, "rotation: dims is even and at most a head's, axes 1 to 4");
    }
    if (r->pos_stride < 0) {
        return refuse(CCK_E_SHAPE, op, "rotation: the positions' stride is negative");
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
    if (r->dims && ((rows && (!r->freq || !r->pos)) || !aligned(r->freq, 4) || !aligned(r->pos, 4))) {
        return refuse(CCK_E_SHAPE, op, "rotation: freq or pos is null or not aligned");
    }
    return CCK_OK;
}
int check_cache(const char* op, const cck_cache* c) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) {
        return refuse(CCK_E_SHAPE, op, "the cache or a part of it is null");
    }
    if (c->pages < 1 || c->heads < 1 || c->heads > kMostHeads) {
        return refuse(CCK_E_SHAPE, op, "the cache has no pages, no heads or more than 65536");
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
    if (!b || (b->sequences && (!b->first || !b->len || !b->table)) || !aligned(b->first, 4) || !aligned(b->len, 4) || !aligned(b->table, 4)) {
        return refuse(CCK_E_SHAPE, op, "the batch or an array of it is null or not aligned");
    }
    if (b->sequences < 0 || b->rows < 0 || b->max_new < 0 || b->max_len < 0 || b->table_pages < 1 || b->table_stride < 0) {
        return refuse(CCK_E_SHAPE, op, "a size of the batch is negative, or its table has no pages");
    }
    if (b->max_len > kMostTokens) {
        return refuse(CCK_E_SHAPE, op, "a sequence has at most 2^30 tokens");
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
// How rows and heads are dealt out to warps, of which a multiprocessor holds 32: whole rows, or parts of a row's heads where rows are few, down to
// one head a lane
RotaryShape rotary_shape(const cck_rotation& r, int rows, int dim, const cck_rows& x, const cck_rows& y, bool inverse, int v, int sms) {
    RotaryShape s{};
    s.dim = dim, s.heads = x.heads, s.sign = inverse ? -1 : 1;
    s.x = x.data, s.y = y.data, s.xr = x.row_stride, s.xh = x.head_stride, s.yr = y.row_stride, s.yh = y.head_stride;
    s.rot_items = r.dims / 2 / v;
    s.items = s.rot_items + (x.data == y.data ? 0 : ceil_div(dim - r.dims, 2 * v));
    if (s.items == 0) { // in place, and nothing turns
        return s;
    }
    const int warps = 32 * sms, at_once = s.items < 32 ? 32 / s.items : 1, most = ceil_div(x.heads, at_once);
    int splits = 1;
    if (rows < warps) {
        splits = ceil_div(warps, rows) < most ? ceil_div(warps, rows) : most;
    } else { // a few rounds of rows: parts of a row where they save a fifth of the rounds
        auto time = [&](int n) { return double((int64_t(rows) * n + warps - 1) / warps) / n; };
        for (int n = 2; n <= 4 && n <= most; n++) {
            splits = time(n) < 0.8 * time(splits) ? n : splits;
        }
    }
    s.part_heads = ceil_div(x.heads, splits);
    s.splits = ceil_div(x.heads, s.part_heads);
    s.units = int64_t(rows) * s.splits;
    return s;
}
// blocks of `threads` that work through it: as many as fit the multiprocessors at once
int64_t rotary_blocks(const RotaryShape& s, int threads, int sms) {
    const int64_t all = (s.units + threads / 32 - 1) / (threads / 32), most = int64_t(32) * sms / (threads / 32);
    return all < most ? all : most;
}
size_t rotary_smem(const cck_rotation& r, int threads) {
    return size_t(threads / 32) * (r.dims / 2) * sizeof(float2);
}

template <class T>
cudaError_t launch_rotary(cudaStream_t st, const cck_rotation& r, const RotaryShape& s, int v, int64_t blocks) {
    auto go = [&](auto kernel) {
        kernel<<<unsigned(blocks), kRotaryThreads, rotary_smem(r, kRotaryThreads), st>>>(r, s);
        return cudaGetLastError();
    };
    constexpr int kMost = 16 / sizeof(T);
    if (r.adjacent) {
        return v == 8 ? go(rotary_kernel<T, kMost, true>) : v == 4 ? go(rotary_kernel<T, 4, true>) : v == 2 ? go(rotary_kernel<T, 2, true>) : go(rotary_kernel<T, 1, true>);
    }
    return v == 8 ? go(rotary_kernel<T, kMost, false>) : v == 4 ? go(rotary_kernel<T, 4, false>) : v == 2 ? go(rotary_kernel<T, 2, false>) : go(rotary_kernel<T, 1, false>);
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
template <class T>
cudaError_t launch_append(cudaStream_t st, const AppendArgs& a, bool pages, int v, unsigned blocks, size_t smem) {
    const int threads = pages && a.group_threads > kAppendThreads ? a.group_threads : kAppendThreads;
    auto go = [&](auto kernel, std::atomic<bool>* ready) {
        if (smem > 47 * 1024) { // 48 with the kernel's own arrays
            if (cudaError_t e = allow_shared(kernel, kAppendSmem, ready)) {
                return e;
            }
        }
        kernel<<<blocks, threads, smem, st>>>(a);
        return cudaGetLastError();
    };
    static std::atomic<bool> ready[11][kMaxDevices];
    if constexpr (sizeof(T) == 2) {
        auto of_dim = [&](auto adjacent) {
            constexpr bool adj = decltype(adjacent)::value;
            switch (a.cache.dim) {
            case 32: return go(append_pages_kernel<T, 32, adj>, ready[3 + adj]);
            case 64: return go(append_pages_kernel<T, 64, adj>, ready[5 + adj]);
            case 96: return go(append_pages_kernel<T, 96, adj>, ready[7 + adj]);
            default: return go(append_pages_kernel<T, 128, adj>, ready[9 + adj]);
            }
        };
        if (pages) {
            const cudaError_t e = a.rotation.adjacent ? of_dim(std::true_type{}) : of_dim(std::false_type{});
            if (e || !a.apart) {
                return e;
            }
            cudaLaunchConfig_t cfg{};
            cudaLaunchAttribute beside;
            beside.id = cudaLaunchAttributeProgrammaticStreamSerialization;
            beside.val.programmaticStreamSerializationAllowed = 1;
            cfg.gridDim = dim3(a.apart), cfg.blockDim = dim3(kRotaryThreads), cfg.dynamicSmemBytes = rotary_smem(a.rotation, kRotaryThreads), cfg.stream = st;
            cfg.attrs = &beside, cfg.numAttrs = 1;
            return a.rotation.adjacent ? cudaLaunchKernelEx(&cfg, query_kernel<T, true>, a) : cudaLaunchKernelEx(&cfg, query_kernel<T, false>, a);
        }
    }
    switch (v) { // vectors of 8 queries go with append_pages_kernel
    case 4: return go(append_kernel<T, 4>, ready[2]);
    case 2: return go(append_kernel<T, 2>, ready[1]);
    default: return go(append_kernel<T, 1>, ready[0]);
    }
}

// How an attention call is cut up: whole units, a block each, or equal shares of the line of all units
struct Plan {
    int nt;                 // tiles of 8 rows of a warp of decode_kernel; 0: tile_kernel
    int granule, tile_rows; // keys and rows of a step
    int row_tiles;          // of a sequence
    int64_t blocks;
    bool shares;
    unsigned merge_x, merge_y; // units that can be split; blocks for the rows of one
    size_t part_bytes, ml_bytes, bytes; // of the workspace
};
Plan make_plan(const cck_cache& c, const cck_batch& b, int q_heads, int sms) {
    Plan p{};
    const int64_t rows = int64_t(b.max_new < b.rows ? b.max_new : b.rows) * (q_heads / c.heads);
    // up to 24 rows by warps of their own, 17 and more in two passes over the keys, the second from L2: 49 | 54 us against the tile kernel at 20 rows, 62 | 54 at
    // 32 (16 sequences of up to 4096, 8 heads of 128)
    p.nt = rows <= 8 ? 1 : rows <= 24 ? 2 : 0;
    p.granule = p.nt ? granule_of(c.dim) : kTileKeys, p.tile_rows = p.nt ? 8 * p.nt : kUnitRows;
    const int64_t row_tiles = (rows + p.tile_rows - 1) / p.tile_rows, tiles = b.sequences * row_tiles; // below 2^31 * 2^43 / 2^3
    if (rows > kMostTokens || tiles * c.heads > 0x7fffffff) {
        p.blocks = int64_t(1) << 32; // refused
        return p;
    }
    p.row_tiles = int(row_tiles);
    const int64_t units = tiles * c.heads, slots = (p.nt == 0 ? 1 : p.nt == 1 ? 3 : 2) * sms;
    const int64_t granules = int64_t(b.max_len) / p.granule + 2;
    const int least = p.nt ? 2 * kDecodeWarps : 2; // granules of a share
    // Shares cost a launch and the way through the workspace, whole units leave multiprocessors idle. us whole | in shares, 8 heads of 128, one token: 1000 keys
    // 13 | 16, 1500 15 | 15, 3000 27 | 15; 64 sequences of 700 29 | 32, of 2048 52 | 48; 256 rows: 512 keys 23 | 28, 1024 25 | 25. Of very many units the
    // last ones hardly show (1000 sequences of 2048: 511 | 549).
    p.shares = granules > (p.nt ? 6 : 5) * least && units < 8 * slots;
    const int64_t most = (units * granules + least - 1) / least;
    p.blocks = !p.shares ? units : most < slots ? most : slots;
    p.blocks = p.shares && p.blocks > kMostShares ? kMostShares : p.blocks;
    if (p.shares) {
        p.merge_x = unsigned(units < p.blocks ? units : p.blocks), p.merge_y = p.nt == 0 ? 16 : p.merge_x < 64 ? p.tile_rows : 1;
        p.part_bytes = size_t(2 * p.blocks) * p.tile_rows * c.dim * 4;
        p.ml_bytes = size_t(2 * p.blocks) * p.tile_rows * 8;
        p.bytes = p.part_bytes + p.ml_bytes + size_t(p.blocks) * sizeof(Split);
    }
    return p;
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
    cfg.gridDim = dim3(p.merge_x, p.merge_y), cfg.blockDim = dim3(kMergeWarps * 32), cfg.stream = st, cfg.attrs = &dependent, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, merge_kernel<T>, a, int(p.blocks));
}

} // namespace

extern "C" {

int cck_rotary(void* stream, const cck_rotation* rotation, int rows, int dim, const cck_rows* x, const cck_rows* y, int inverse) {
    const char* op = "cck_rotary";
    if (!rotation || rows < 0 || dim < 1 || dim > 1024) {
        return refuse(CCK_E_SHAPE, op, "rotation is null, rows is negative or dim is not 1 to 1024");
    }
    int e;
    if ((e = check_rotation(op, rotation, rows, dim)) || (e = check_rows(op, x, "x", rows, 0, true)) || (e = check_rows(op, y, "y", rows, 0, true)) || (e = check_pair(op, x, y, rows, dim))) {
        return e;
    }
    int sms = 0;
    if ((e = device_of(op, {x->data, y->data, rotation->dims ? rotation->freq : nullptr, rotation->dims ? rotation->pos : nullptr}, sms))) {
        return e;
    }
    if (rows == 0) {
        return CCK_OK;
    }
    const int v = rotary_vector(*rotation, dim, *x, *y);
    const RotaryShape s = rotary_shape(*rotation, rows, dim, *x, *y, inverse != 0, v, sms);
    const int64_t blocks = rotary_blocks(s, kRotaryThreads, sms);
    if (blocks == 0) {
        return CCK_OK;
    }
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (x->dtype) {
    case CCK_BF16: return launched(op, launch_rotary<__nv_bfloat16>(st, *rotation, s, v, blocks));
    case CCK_F16: return launched(op, launch_rotary<__half>(st, *rotation, s, v, blocks));
    default: return launched(op, launch_rotary<float>(st, *rotation, s, v, blocks));
    }
}

int cck_cache_append(void* stream, const cck_cache* cache, const cck_batch* batch, const cck_rows* k, const cck_rows* v, const cck_rotation* rotation, const cck_rows* q,
                     const cck_rows* q_out, int32_t* status) {
    const char* op = "cck_cache_append";
    int e;
    if ((e = check_cache(op, cache)) || (e = check_batch(op, batch)) || (e = check_rows(op, k, "k", batch->rows, 16, true)) ||
        (e = check_rows(op, v, "v", batch->rows, 16, true))) {
        return e;
    }
    if (k->dtype != v->dtype || k->heads != cache->heads || v->heads != cache->heads) {
        return refuse(CCK_E_SHAPE, op, "k and v have the cache's heads and one type");
    }
    if (rotation && (e = check_rotation(op, rotation, batch->rows, cache->dim))) {
        return e;
    }
    if (q) {
        if (!rotation) {
            return refuse(CCK_E_SHAPE, op, "queries are rotated, but there is no rotation");
        }
        if ((e = check_rows(op, q, "q", batch->rows, 0, true)) || (e = check_rows(op, q_out, "q_out", batch->rows, 0, true)) ||
            (e = check_pair(op, q, q_out, batch->rows, cache->dim))) {
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
    const bool turns = rotation && rotation->dims;
    if ((e = device_of(op, {cache->k, cache->v, cache->k_scale, cache->v_scale, batch->first, batch->len, batch->table, k->data, v->data, turns ? rotation->freq : nullptr,
                            turns ? rotation->pos : nullptr, q ? q->data : nullptr, q ? q_out->data : nullptr, status},
                       sms))) {
        return e;
    }
    AppendArgs a{};
    a.cache = *cache, a.batch = *batch, a.k = k->data, a.v = v->data, a.status = status;
    a.kr = k->row_stride, a.kh = k->head_stride, a.vr = v->row_stride, a.vh = v->head_stride;
    if (rotation) {
        a.rotation = *rotation;
    }
    const int max_new = batch->max_new < batch->rows ? batch->max_new : batch->rows;
    const int P = cache->page_tokens, D = cache->dim, most = max_new < P ? max_new : P; // new rows of a page
    a.batch.max_new = max_new;
    // without room for rows, a block for each sequence still says so if there are any
    a.blocks_per_seq = max_new ? int((int64_t(max_new) + P - 2) / P + 1) : status ? 1 : 0;
    int64_t more = 0;
    int vec = 0;
    size_t smem = 0;
    if (q && batch->rows && batch->sequences) { // without sequences all rows are nobody's
        vec = rotary_vector(*rotation, D, *q, *q_out);
        a.q = rotary_shape(*rotation, batch->rows, D, *q, *q_out, false, vec, sms);
    }
    const int64_t units = int64_t(batch->sequences) * a.blocks_per_seq;
    if (units > 0x7fffffff) {
        return refuse(CCK_E_SHAPE, op, "too many rows for one launch");
    }
    // 16-bit values whose rotated part is whole vectors go through registers
    const bool pages = k->dtype != CCK_F32 && a.rotation.dims % 16 == 0 && (vec == 0 || vec == 8);
    int64_t kv;
    if (pages) {
        // threads of a (page, head): the fewest whose items cover the new rows; then blocks for a page's heads, as long as multiprocessors are
        // left for them, or three each where a page's angles, which each computes anew, are few (1, 2, 4, 8 blocks a multiprocessor: 27, 37, 35,
        // 44 us for the keys and values of eight prompts, 64 tokens of 64 pairs a page; 1, 2: 16.5, 14.5 us for 16 tokens of 32 pairs)
        const int groups = (most + 14) / 16 + 1 < P / 16 ? (most + 14) / 16 + 1 : P / 16;
        a.group_threads = 32;
        while (most * (D / 16) > kKeyItems * a.group_threads || groups * (D / 2) > kValueItems * a.group_threads) {
            a.group_threads *= 2;
        }
        const int passes = ceil_div(cache->heads, a.group_threads < kAppendThreads ? kAppendThreads / a.group_threads : 1);
        const int angles = most * (a.rotation.dims / 2) / kAppendThreads; // of a thread
        const int64_t want = units ? ((angles > 4 ? 1 : 3) * int64_t(sms) + units - 1) / units : 1;
        a.head_splits = int(want < passes ? want : passes);
        kv = units * a.head_splits;
        const size_t table = size_t(most) * (a.rotation.dims / 2) * sizeof(float2);
        smem = table > smem ? table : smem;
    } else {
        kv = units * cache->heads;
        const size_t rows = append_smem(most, D, size_of(k->dtype));
        smem = rows > smem ? rows : smem;
    }
    if (vec && pages && units && batch->rows >= 32 * sms) {
        // a launch of their own for queries that fill the GPU: 55 -> 49 us for eight prompts of about 900 tokens, 32 heads of 128; with 2000 rows of
        // 20 heads of 64 it took 19 us instead of 16
        a.apart = int(rotary_blocks(a.q, kRotaryThreads, sms));
    }
    if (vec && !a.apart) {
        const int threads = pages && a.group_threads > kAppendThreads ? a.group_threads : kAppendThreads;
        more = rotary_blocks(a.q, threads, sms);
        smem = more && rotary_smem(*rotation, threads) > smem ? rotary_smem(*rotation, threads) : smem;
    }
    if (kv + more > 0x7fffffff) {
        return refuse(CCK_E_SHAPE, op, "too many rows for one launch");
    }
    a.kv_blocks = int(kv);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (kv + more == 0) {
        return CCK_OK;
    }
    const unsigned blocks = unsigned(kv + more);
    switch (k->dtype) {
    case CCK_BF16: return launched(op, launch_append<__nv_bfloat16>(st, a, pages, vec, blocks, smem));
    case CCK_F16: return launched(op, launch_append<__half>(st, a, pages, vec, blocks, smem));
    default: return launched(op, launch_append<float>(st, a, false, vec, blocks, smem));
    }
}

size_t cck_cache_attention_workspace_bytes(const cck_cache* cache, const cck_batch* batch, int q_heads) {
    const char* op = "cck_cache_attention_workspace_bytes";
    int sms = 0;
    if (check_cache(op, cache) || check_batch(op, batch) || q_heads < 1 || q_heads > kMostHeads || q_heads % cache->heads || device_of(op, {}, sms)) {
        return 0;
    }
    return make_plan(*cache, *batch, q_heads, sms).bytes;
}

int cck_cache_attention(void* stream, const cck_cache* cache, const cck_batch* batch, const cck_rows* q, const cck_rows* out, float* lse, float softmax_scale, int causal,
                        int window, void* ws, size_t ws_bytes) {
    const char* op = "cck_cache_attention";
    int e;
    if ((e = check_cache(op, cache)) || (e = check_batch(op, batch)) || (e = check_rows(op, q, "q", batch->rows, 16, false)) ||
        (e = check_rows(op, out, "out", batch->rows, 16, false)) ||
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
    if ((e = device_of(op, {cache->k, cache->v, cache->k_scale, cache->v_scale, batch->first, batch->len, batch->table, q->data, out->data, lse}, sms))) {
        return e;
    }
    if (batch->sequences == 0 || batch->rows == 0 || batch->max_new == 0) {
        return CCK_OK;
    }
    const Plan p = make_plan(*cache, *batch, q->heads, sms);
    if (p.blocks > 0x7fffffff) {
        return refuse(CCK_E_SHAPE, op, "too many rows for one launch");
    }
    if (ws_bytes < p.bytes || (p.bytes && (!ws || !aligned(ws, 16)))) {
        return refuse(CCK_E_WORKSPACE, op, "the workspace is too small, null or not aligned");
    }
    if (p.bytes && (e = device_of(op, {ws}, sms))) {
        return e;
    }
    AttentionArgs a{};
    a.cache = *cache, a.batch = *batch, a.q = q->data, a.out = out->data, a.lse = lse;
    a.qr = q->row_stride, a.qh = q->head_stride, a.or_ = out->row_stride, a.oh = out->head_stride;
    a.scale_log2 = softmax_scale * 1.4426950408889634f;
    a.q_heads = q->heads, a.group = q->heads / cache->heads, a.causal = causal != 0, a.window = window;
    const int64_t reach = int64_t(batch->table_pages) * cache->page_tokens;
    a.reach = int(reach < kMostTokens ? reach : kMostTokens);
    a.granule_shift = __builtin_ctz(p.granule), a.unit_cost = p.nt ? 8 : 3, a.page_shift = __builtin_ctz(cache->page_tokens);
    a.tile_rows = p.tile_rows, a.row_tiles = p.row_tiles, a.lose = g_lose.load(std::memory_order_relaxed);
    if (p.shares) {
        a.part_o = static_cast<float*>(ws), a.part_ml = reinterpret_cast<float*>(static_cast<char*>(ws) + p.part_bytes);
        a.splits = reinterpret_cast<Split*>(static_cast<char*>(ws) + p.part_bytes + p.ml_bytes);
    }
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return launched(op, q->dtype == CCK_BF16 ? launch_attention<__nv_bfloat16>(st, a, p) : launch_attention<__half>(st, a, p));
}

void cck_set_lost_copy_test(int block) {
    g_lose.store(block, std::memory_order_relaxed);
}

} // extern "C"
