// Key/value cache operators for sm_100a, host side: argument checks and
// launches of q4rdna_kv_append.cuh, q4rdna_kv_attention.cuh and q4rdna_kv_tile.cuh.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <map>
#include <mutex>
#include <set>

#include "q4rdna_kv.h"
#include "q4rdna_kv_append.cuh"
#include "q4rdna_kv_attention.cuh"
#include "q4rdna_kv_tile.cuh"

namespace q4 {
extern std::atomic<uint64_t> g_launches;  // q4rdna_gemv.cu: kernels launched by the library
}

namespace q4kv {

bool aligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int type_bytes(int type) { return type == Q4RDNA_F32 ? 4 : 2; }

q4rdna_status check_cache(const q4rdna_kv_cache *c, Cache &out) {
    if (c == nullptr || c->tiles == nullptr) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (c->pages <= 0 || c->kv_heads <= 0) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (c->format != Q4RDNA_KV_INT8 && c->format != Q4RDNA_KV_E4M3) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (q4rdna_kv_cache_bytes(c) == 0) return Q4RDNA_ERR_SHAPE;
    if (!aligned(c->tiles)) return Q4RDNA_ERR_ALIGNMENT;
    out.tiles = c->tiles;
    out.pages = c->pages;
    out.hk = c->kv_heads;
    out.nbl = 0;
    while ((kBlock << out.nbl) < c->page_tokens) ++out.nbl;
    out.format = c->format;
    out.tile_bytes = (int)q4rdna_kv_tile_bytes(c->head_dim);
    return Q4RDNA_OK;
}

q4rdna_status check_batch(const q4rdna_kv_cache *c, const q4rdna_kv_batch *b, int tokens, Batch &out) {
    if (b == nullptr) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (b->sequences != 0 && (b->page_table == nullptr || b->lengths == nullptr)) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (b->sequences < 0 || b->table_stride <= 0 || b->max_length < 0 || tokens < 0) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (b->q_start == nullptr && tokens != b->sequences) return Q4RDNA_ERR_SHAPE;
    const long long room = std::min<long long>((long long)b->table_stride * c->page_tokens, kMaxTokens);
    if (b->max_length > room) return Q4RDNA_ERR_SHAPE;
    // the append's units and the attention's 32-bit row arithmetic
    if (b->sequences > (1 << 28) || tokens > (1 << 28)) return Q4RDNA_ERR_TOO_LARGE;
    out.table = b->page_table;
    out.lengths = b->lengths;
    out.q_start = b->q_start;
    out.S = b->sequences;
    out.stride = b->table_stride;
    out.max_len = b->max_length > 0 ? b->max_length : (int)room;
    out.T = tokens;
    return Q4RDNA_OK;
}

// A row operand: [rows][heads][D] with `stride` elements from row to row
q4rdna_status check_rows(const void *p, int64_t stride, int type, int heads, int D) {
    if (p == nullptr) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (stride < (int64_t)heads * D) return Q4RDNA_ERR_SHAPE;
    if (!aligned(p) || stride * type_bytes(type) % 16 != 0) return Q4RDNA_ERR_ALIGNMENT;
    return Q4RDNA_OK;
}

bool known_type(int t) { return t == Q4RDNA_F32 || t == Q4RDNA_F16 || t == Q4RDNA_BF16; }

// One launch as a programmatic dependent of the stream's last kernel: it may be
// set up while that one ends, and every kernel here waits for it
// (griddepcontrol.wait) before its first access.
template <class... Args>
q4rdna_status launch(void (*kernel)(Args...), dim3 grid, int threads, size_t smem, cudaStream_t stream, const Args &...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
        cudaGetLastError();
        return Q4RDNA_ERR_CUDA;
    }
    q4::g_launches.fetch_add(1, std::memory_order_relaxed);
    return Q4RDNA_OK;
}

q4rdna_status launched() {
    if (cudaGetLastError() != cudaSuccess) return Q4RDNA_ERR_CUDA;
    q4::g_launches.fetch_add(1, std::memory_order_relaxed);
    return Q4RDNA_OK;
}

q4rdna_status check_attention(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch,
                              const q4rdna_kv_attention_args *args, AttnArgs &A) {
    q4rdna_status st = check_cache(cache, A.c);
    if (st != Q4RDNA_OK) return st;
    if (args == nullptr || !known_type(args->type) || args->window < 0) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (!std::isfinite(args->scale) || args->scale < 0.0f) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if ((st = check_batch(cache, batch, args->tokens, A.b)) != Q4RDNA_OK) return st;
    if (args->heads <= 0) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (args->heads % cache->kv_heads != 0) return Q4RDNA_ERR_SHAPE;
    const int D = cache->head_dim;
    if (args->tokens > 0) {
        if ((st = check_rows(args->q, args->q_stride, args->type, args->heads, D)) != Q4RDNA_OK) return st;
        if ((st = check_rows(args->out, args->out_stride, args->type, args->heads, D)) != Q4RDNA_OK) return st;
    }
    A.q = args->q;
    A.out = args->out;
    A.qs = args->q_stride;
    A.os = args->out_stride;
    A.type = args->type;
    A.heads = args->heads;
    A.group = args->heads / cache->kv_heads;
    const float scale = args->scale > 0.0f ? args->scale : 1.0f / std::sqrt((float)D);
    A.scale = scale * 1.44269504088896340736f;
    A.window = args->window < A.b.max_len ? args->window : 0;
    if ((long long)args->tokens * A.group > (1 << 30)) return Q4RDNA_ERR_TOO_LARGE;  // columns of a kv head
    return Q4RDNA_OK;
}

struct AppendVariant {
    void (*kernel)(AppendArgs);
    int smem;  // the ring; kTurnPart takes 16 rows more
};
template <int D, int TYPE, int FMT>
AppendVariant append_variant(int turn) {
    constexpr int ring = Ring<D, TYPE>::BYTES;
    if (turn == kTurnHalves) return {kv_append_kernel<D, TYPE, FMT, kTurnHalves>, ring};
    if (turn == kTurnPairs) return {kv_append_kernel<D, TYPE, FMT, kTurnPairs>, ring};
    return {kv_append_kernel<D, TYPE, FMT, kTurnPart>, ring + 16 * (D + 1) * (int)sizeof(float)};
}
template <int D, int TYPE>
AppendVariant append_variant(int format, int turn) {
    return format == Q4RDNA_KV_INT8 ? append_variant<D, TYPE, Q4RDNA_KV_INT8>(turn)
                                    : append_variant<D, TYPE, Q4RDNA_KV_E4M3>(turn);
}
template <int D>
AppendVariant append_variant(int type, int format, int turn) {
    if (type == Q4RDNA_F32) return append_variant<D, Q4RDNA_F32>(format, turn);
    if (type == Q4RDNA_F16) return append_variant<D, Q4RDNA_F16>(format, turn);
    return append_variant<D, Q4RDNA_BF16>(format, turn);
}

// Raises a kernel's shared-memory limit, once per device
bool raise_smem(const void *kernel, int bytes) try {
    static std::mutex mu;
    static std::set<std::pair<int, const void *>> done;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    std::lock_guard<std::mutex> lock(mu);
    if (done.count({dev, kernel})) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    done.insert({dev, kernel});
    return true;
} catch (...) {  // out of memory: nothing may be thrown through the C functions
    return false;
}

// ---- the attention's launches

using AttnKernel = void (*)(AttnArgs);

struct Variant {
    AttnKernel kernel;
    size_t smem;
    int threads, nc, shift;  // columns of a task, log2 of the tokens of a piece
};

template <int D, int FMT, int NT, int TERMS>
Variant variant() {
    return {kv_attention_kernel<D, FMT, NT, TERMS>, sizeof(AttnSmem<D, NT>), kAttnThreads, 8 * NT, 4};
}
template <int D, int FMT>
Variant variant(int nt, int terms) {
    if (nt == 1) return terms == 1 ? variant<D, FMT, 1, 1>() : variant<D, FMT, 1, 2>();
    return terms == 1 ? variant<D, FMT, 2, 1>() : variant<D, FMT, 2, 2>();
}
template <int D>
Variant variant(int format, int nt, int terms) {
    return format == Q4RDNA_KV_INT8 ? variant<D, Q4RDNA_KV_INT8>(nt, terms) : variant<D, Q4RDNA_KV_E4M3>(nt, terms);
}
template <int D>
Variant tile32_variant(int format) {
    return {format == Q4RDNA_KV_INT8 ? kv_tile32_kernel<D, Q4RDNA_KV_INT8> : kv_tile32_kernel<D, Q4RDNA_KV_E4M3>,
            sizeof(TileSmem<D>), kTileThreads, kTile32Cols, kTileShift};
}
template <int D>
Variant tile_variant(int format) {
    return {format == Q4RDNA_KV_INT8 ? kv_tile_kernel<D, Q4RDNA_KV_INT8> : kv_tile_kernel<D, Q4RDNA_KV_E4M3>,
            sizeof(TileSmem<D>), kTileThreads, kTileCols, kTileShift};
}

// One of the attention's kernels with its part of the workspace
struct AttnLaunch {
    Variant v;
    unsigned grid;  // CTAs, one share each
    int few, many;  // columns of the sequences that it takes
    int min_share;
    size_t workspace;
};

// CTAs of the kernel that the current device holds at once (its shared-memory limit raised); 0 on an error
int resident_ctas(const Variant &v) try {
    static std::mutex mu;
    static std::map<std::pair<int, AttnKernel>, int> known;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    std::lock_guard<std::mutex> lock(mu);
    int &n = known[{dev, v.kernel}];
    if (n == 0) {
        int sms = 0, occ = 0;
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
            cudaFuncSetAttribute(v.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)v.smem) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, v.kernel, v.threads, v.smem) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        n = sms * std::max(occ, 1);
    }
    return n;
} catch (...) {
    return 0;
}

q4rdna_status size_launch(const AttnArgs &A, int D, AttnLaunch &L) {
    const int ctas = resident_ctas(L.v);
    if (ctas == 0) return Q4RDNA_ERR_DEVICE;
    // no more CTAs than the largest work has shares
    const double tasks = ((double)A.b.T * A.group / L.v.nc + A.b.S) * A.c.hk;
    const double work = tasks * ((A.b.max_len >> L.v.shift) + 1);
    L.grid = (unsigned)std::max(1.0, std::min((double)ctas, work / L.min_share + 1.0));
    L.workspace = (size_t)L.grid * (2 * sizeof(int4) + 2 * sizeof(float) * part_floats(D, L.v.nc));
    return Q4RDNA_OK;
}

// Columns (new tokens x query heads of a kv head) from which on the tile kernels take a
// sequence.  Measured with 32 query and 8 kv heads of 128, int8, us for the kernel for few
// columns and for the tile kernel (sequences x tokens):
//   columns               16       64       96      128      256       512
//   f32   1 x 64      10, 29   13, 31   19, 34   20, 37   34, 37
//         1 x 512     11, 23   13, 25   18, 27   19, 29   24, 30    33, 30
//         1 x 4096    17, 32   26, 34   32, 36   37, 38   60, 40   105, 63
//         1 x 16384   26, 59   57, 64   78, 67   99, 70  184, 92  353, 143
//         4 x 4096    27, 52   60, 56   86, 59  106, 63  196, 88  370, 145
//   bf16  1 x 64      10, 24   13, 26   19, 27   19, 29   33, 37
//         1 x 512     10, 22   12, 24   18, 24   18, 26   23, 31    30, 32
//         1 x 4096    16, 31   24, 33   29, 34   33, 35   52, 41    91, 42
//         1 x 16384   24, 53   49, 57   67, 59   84, 60  155, 73   294, 90
//         4 x 4096    25, 47   53, 50   74, 52   91, 53  166, 68   312, 94
// The rule knows the columns only: with 500 tokens or fewer the kernel for few columns is
// faster up to 256 columns, by 17 us at most.
constexpr int kTileFrom = 96;

// The launches of a call: sequences of few columns, sequences of many, or both
q4rdna_status plan_attention(const AttnArgs &A, int D, AttnLaunch (&L)[2], int &n) {
    n = 0;
    const long long most = A.b.q_start == nullptr ? A.group : (long long)A.b.T * A.group;  // columns of a sequence
    const bool f32 = A.type == Q4RDNA_F32;
    const bool tiles = D <= 128 && most >= kTileFrom;
    // One sequence, or a few of many columns on average, no length more than twice the average of the new tokens: no
    // launches for sequences of few columns, which the tile kernels take too.  us for the tile kernel alone and for both
    // (32 / 8 heads of 128):
    //                              bf16          f32
    //   2 x 300, 4 x 300      48, 52   50, 55          72, 77 (4 x 300)
    //   400 and 1 of 400          47, 59       43, 55
    //   3000 and 1 of 3000     277, 293     508, 519
    //   400 and 3 of 8191       122, 73      152, 72     (beyond the bound on the lengths)
    //   400 and 3 of 65521     728, 177     788, 193
    const bool alone = A.b.S == 1 || A.b.q_start == nullptr ||
                       (A.b.S <= 4 && most >= 4LL * kTileFrom * A.b.S && (long long)A.b.max_len * A.b.S <= 2LL * A.b.T);
    if (!tiles || !alone) {
        // One column tile (two CTAs an SM; a sequence of more columns has several tasks) or two, us for 16 sequences of
        // 4001 tokens, 8 kv heads, f32:
        //   columns             8       16       32
        //   head_dim 128   37, 50   55, 56   74, 79
        //   head_dim 256   56, 83   92, 99  131, 139   (4 kv heads, 9664 columns, 604 tokens: 954, 831)
        const int nt = (long long)A.b.T * A.group <= 32LL * A.b.S ? 1 : 2, terms = A.type == Q4RDNA_F32 ? 2 : 1;
        AttnLaunch &l = L[n++];
        l.v = D == 64 ? variant<64>(A.c.format, nt, terms)
                      : D == 128 ? variant<128>(A.c.format, nt, terms) : variant<256>(A.c.format, nt, terms);
        l.few = 0;
        l.many = tiles ? kTileFrom : INT_MAX;
        l.min_share = kAttnWarps;  // one block per warp
    }
    if (tiles) {
        AttnLaunch &l = L[n++];
        if (f32) l.v = D == 64 ? tile32_variant<64>(A.c.format) : tile32_variant<128>(A.c.format);
        else l.v = D == 64 ? tile_variant<64>(A.c.format) : tile_variant<128>(A.c.format);
        l.few = n == 2 ? kTileFrom : 0;
        l.many = INT_MAX;
        l.min_share = 2;
    }
    for (int i = 0; i < n; ++i) {
        const q4rdna_status st = size_launch(A, D, L[i]);
        if (st != Q4RDNA_OK) return st;
    }
    return Q4RDNA_OK;
}

}  // namespace q4kv

uint32_t q4kv_take_fault() {
    unsigned v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, q4kv::g_kv_fault, sizeof(v)) != cudaSuccess) return 0xffffffffu;
    if (v != 0) cudaMemcpyToSymbol(q4kv::g_kv_fault, &zero, sizeof(zero));
    return v;
}

extern "C" {

size_t q4rdna_kv_tile_bytes(int head_dim) {
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
    return q4kv::kHeader + 2 * (size_t)q4kv::kBlock * head_dim;
}

size_t q4rdna_kv_cache_bytes(const q4rdna_kv_cache *c) {
    if (c == nullptr || c->pages <= 0 || c->kv_heads <= 0) return 0;
    const int p = c->page_tokens;
    if (p < 16 || p > 256 || (p & (p - 1)) != 0) return 0;
    return (size_t)c->pages * c->kv_heads * (p / q4kv::kBlock) * q4rdna_kv_tile_bytes(c->head_dim);
}

q4rdna_status q4rdna_kv_append(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch,
                               const q4rdna_kv_append_args *args, q4rdna_stream_t stream) {
    using namespace q4kv;
    AppendArgs A{};
    q4rdna_status st = check_cache(cache, A.c);
    if (st != Q4RDNA_OK) return st;
    if (args == nullptr || !known_type(args->type) || args->heads < 0) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if ((args->q_norm != nullptr || args->k_norm != nullptr) && (!std::isfinite(args->norm_eps) || args->norm_eps < 0.0f))
        return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (args->rope != Q4RDNA_ROPE_NEOX && args->rope != Q4RDNA_ROPE_NORM) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if ((st = check_batch(cache, batch, args->tokens, A.b)) != Q4RDNA_OK) return st;
    const int D = cache->head_dim;
    const int rot = args->inv_freq == nullptr ? 0 : args->rotary_dim == 0 ? D : args->rotary_dim;
    if (rot < 0 || rot > D || rot % 16 != 0) return Q4RDNA_ERR_SHAPE;
    if (args->heads % cache->kv_heads != 0) return Q4RDNA_ERR_SHAPE;
    if (!aligned(args->q_norm) || !aligned(args->k_norm)) return Q4RDNA_ERR_ALIGNMENT;
    if (args->tokens > 0) {
        if ((st = check_rows(args->k, args->k_stride, args->type, cache->kv_heads, D)) != Q4RDNA_OK) return st;
        if ((st = check_rows(args->v, args->v_stride, args->type, cache->kv_heads, D)) != Q4RDNA_OK) return st;
        if (args->heads > 0) {
            if ((st = check_rows(args->q, args->q_stride, args->type, args->heads, D)) != Q4RDNA_OK) return st;
            if ((st = check_rows(args->q_out, args->q_out_stride, args->type, args->heads, D)) != Q4RDNA_OK) return st;
        }
    }
    if (args->tokens == 0 || batch->sequences == 0) return Q4RDNA_OK;
    A.k = args->k; A.v = args->v; A.q = args->q; A.q_out = args->q_out;
    A.ks = args->k_stride; A.vs = args->v_stride; A.qs = args->q_stride; A.qos = args->q_out_stride;
    A.inv_freq = args->inv_freq; A.q_norm = args->q_norm; A.k_norm = args->k_norm; A.positions = args->positions;
    A.heads = args->heads; A.rot = rot;
    A.eps = args->norm_eps;
    const int units = batch->q_start == nullptr ? batch->sequences : args->tokens / kBlock + 2 * batch->sequences;
    // Heads of a block over several CTAs where the blocks alone would not fill the GPU (each CTA makes the
    // block's cosines anew): about 4 CTAs per SM
    const int slices = std::max(1, std::min(std::min(cache->kv_heads, 65535), (4 * 148 + units - 1) / units));
    const int turn = rot == 0 || (args->rope == Q4RDNA_ROPE_NEOX && rot == D) ? kTurnHalves
                     : args->rope == Q4RDNA_ROPE_NORM                         ? kTurnPairs
                                                                              : kTurnPart;
    const int f = cache->format;
    const AppendVariant v = D == 64 ? append_variant<64>(args->type, f, turn)
                                    : D == 128 ? append_variant<128>(args->type, f, turn) : append_variant<256>(args->type, f, turn);
    if (!raise_smem((const void *)v.kernel, v.smem)) return Q4RDNA_ERR_DEVICE;
    return launch(v.kernel, dim3((unsigned)units, (unsigned)slices), D, v.smem, (cudaStream_t)stream, A);
}

q4rdna_status q4rdna_kv_dequant(const q4rdna_kv_cache *cache, const int32_t *page_list, int count, int type, void *k,
                                void *v, q4rdna_stream_t stream) {
    using namespace q4kv;
    Cache c{};
    const q4rdna_status st = check_cache(cache, c);
    if (st != Q4RDNA_OK) return st;
    if (count < 0 || !known_type(type)) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (count == 0) return Q4RDNA_OK;
    if (page_list == nullptr || k == nullptr || v == nullptr) return Q4RDNA_ERR_INVALID_ARGUMENT;
    if (!aligned(k) || !aligned(v)) return Q4RDNA_ERR_ALIGNMENT;
    const long long n = ((long long)count * c.hk) << c.nbl;
    if (n > 0x7fffffffLL) return Q4RDNA_ERR_TOO_LARGE;
    const cudaStream_t cs = (cudaStream_t)stream;
    if (cache->head_dim == 64) kv_dequant_kernel<64><<<(unsigned)n, 128, 0, cs>>>(c, page_list, type, k, v);
    else if (cache->head_dim == 128) kv_dequant_kernel<128><<<(unsigned)n, 128, 0, cs>>>(c, page_list, type, k, v);
    else kv_dequant_kernel<256><<<(unsigned)n, 128, 0, cs>>>(c, page_list, type, k, v);
    return launched();
}

size_t q4rdna_kv_attention_workspace_bytes(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch,
                                           const q4rdna_kv_attention_args *args) {
    using namespace q4kv;
    AttnArgs A{};
    AttnLaunch L[2];
    int n = 0;
    if (check_attention(cache, batch, args, A) != Q4RDNA_OK || args->tokens == 0 || batch->sequences == 0) return 0;
    if (plan_attention(A, cache->head_dim, L, n) != Q4RDNA_OK) return 0;
    size_t bytes = 0;
    for (int i = 0; i < n; ++i) bytes += L[i].workspace;
    return bytes;
}

q4rdna_status q4rdna_kv_attention(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch,
                                  const q4rdna_kv_attention_args *args, void *workspace, size_t workspace_bytes,
                                  q4rdna_stream_t stream) {
    using namespace q4kv;
    AttnArgs A{};
    AttnLaunch L[2];
    int n = 0;
    q4rdna_status st = check_attention(cache, batch, args, A);
    if (st != Q4RDNA_OK) return st;
    if (args->tokens == 0 || batch->sequences == 0) return Q4RDNA_OK;
    const int D = cache->head_dim;
    if ((st = plan_attention(A, D, L, n)) != Q4RDNA_OK) return st;
    size_t bytes = 0;
    for (int i = 0; i < n; ++i) bytes += L[i].workspace;
    if (workspace == nullptr || workspace_bytes < bytes) return Q4RDNA_ERR_WORKSPACE;
    if (!aligned(workspace)) return Q4RDNA_ERR_ALIGNMENT;
    const cudaStream_t cs = (cudaStream_t)stream;
    uint8_t *at = reinterpret_cast<uint8_t *>(workspace);
    for (int i = 0; i < n; ++i) {
        const AttnLaunch &l = L[i];
        A.few = l.few;
        A.many = l.many;
        A.min_share = l.min_share;
        A.rec = reinterpret_cast<int4 *>(at);
        A.part = reinterpret_cast<float *>(A.rec + 2 * l.grid);
        at += l.workspace;
        if ((st = launch(l.v.kernel, dim3(l.grid), l.v.threads, l.v.smem, cs, A)) != Q4RDNA_OK) return st;
        const bool wide = l.v.nc > 16;
        const auto join = wide ? (D == 64 ? kv_join_wide_kernel<64> : kv_join_wide_kernel<128>)
                               : (D == 64 ? kv_join_kernel<64> : D == 128 ? kv_join_kernel<128> : kv_join_kernel<256>);
        const unsigned y = (unsigned)(wide ? l.v.nc / (kJoinWarps * kJoinCols) : l.v.nc);
        if ((st = launch(join, dim3(l.grid, y), 32 * kJoinWarps, 0, cs, A, l.v.nc)) != Q4RDNA_OK) return st;
    }
    return Q4RDNA_OK;
}

}  // extern "C"
