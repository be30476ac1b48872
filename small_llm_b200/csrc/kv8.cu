// C ABI of the 8-bit paged KV cache (include/sllm.h): checks of arguments and launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>

#include "../../include/sllm.h"
#include "abi.cuh"
#include "attn_kv8.cuh"
#include "attn_kv8_tc.cuh"
#include "kv8.cuh"

using namespace sllm;

namespace {

constexpr int kMaxDev = 64;

int cuda_fail(cudaError_t err, const char* what) {
    char b[256];
    std::snprintf(b, sizeof b, "%s: CUDA error %s: %s", what, cudaGetErrorName(err), cudaGetErrorString(err));
    return fail_text(SLLM_ERR_CUDA, b);
}
int bad(const char* what, const char* why) {
    char b[256];
    std::snprintf(b, sizeof b, "%s: %s", what, why);
    return fail_text(SLLM_ERR_INVALID, b);
}

// The current device and its SM count, which is looked up once.
int current_device(const char* what, int* dev, int* sms) {
    static std::atomic<int> known[kMaxDev];          // SM count, 0 = not looked up
    if (cudaError_t err = cudaGetDevice(dev)) { (void)cudaGetLastError(); return cuda_fail(err, what); }
    if (*dev < 0 || *dev >= kMaxDev) return bad(what, "device ordinal out of range");
    int n = known[*dev].load(std::memory_order_relaxed);
    if (n == 0) {
        int major = 0;
        cudaError_t err = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, *dev);
        if (!err) err = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *dev);
        if (err) return cuda_fail(err, what);
        if (major != 10) { char b[128]; std::snprintf(b, sizeof b, "%s: needs a device of compute capability 10.x", what); return fail_text(SLLM_ERR_CUDA, b); }
        known[*dev].store(n, std::memory_order_relaxed);
    }
    *sms = n;
    return SLLM_OK;
}

// A pointer that a kernel would read or write must belong to the device the kernel runs on.
int check_memory(const char* what, int dev, std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs) {
        if (!p) continue;
        cudaPointerAttributes at{};
        if (cudaError_t err = cudaPointerGetAttributes(&at, p)) { (void)cudaGetLastError(); return cuda_fail(err, what); }
        if ((at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) || (at.type == cudaMemoryTypeDevice && at.device != dev))
            return bad(what, "a pointer is not memory of the current device");
    }
    return SLLM_OK;
}
bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check_layer(const char* what, const sllm_kv8_layer* c) {
    if (!c || !c->pages || !c->scales) return bad(what, "null cache pointer");
    if (c->head_dim != 16 && c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128) return bad(what, "head_dim must be 16, 32, 64 or 128");
    if (c->kv_heads < 1 || c->kv_heads > 1024) return bad(what, "kv_heads must be 1..1024");
    if (c->n_pages < 1 || c->n_pages > 0x7fffffffull) return bad(what, "n_pages must be 1..2^31 - 1");
    if (!aligned(c->pages, 16) || !aligned(c->scales, 16)) return bad(what, "pages and scales must be 16-byte aligned");
    return SLLM_OK;
}
Kv8View view(const sllm_kv8_layer* c) { return Kv8View{c->pages, c->scales, (long long)c->n_pages, (int)c->kv_heads}; }

// Every kernel here starts with griddepcontrol.wait, so it may be scheduled while the stream's previous kernel drains.
template <typename... K, typename... A>
int launch_cluster(const char* what, void (*kern)(K...), dim3 grid, int block, size_t smem, void* stream, unsigned cluster_z, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid; cfg.blockDim = dim3(block); cfg.dynamicSmemBytes = smem; cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = cluster_z;
    cfg.attrs = attr; cfg.numAttrs = cluster_z > 1 ? 2 : 1;
    if (cudaError_t err = cudaLaunchKernelEx(&cfg, kern, args...)) { (void)cudaGetLastError(); return cuda_fail(err, what); }
    return SLLM_OK;
}
template <typename... K, typename... A>
int launch(const char* what, void (*kern)(K...), dim3 grid, int block, size_t smem, void* stream, A... args) {
    return launch_cluster(what, kern, grid, block, smem, stream, 1, args...);
}
// Shared memory above 48 KB, asked for once per kernel and device.
template <typename K>
int opt_in(const char* what, K kern, size_t smem, int dev, std::atomic<uint64_t>& done) {
    const uint64_t bit = 1ull << dev;
    if (smem <= 48 * 1024 || (done.load(std::memory_order_relaxed) & bit)) return SLLM_OK;
    if (cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) { (void)cudaGetLastError(); return cuda_fail(err, what); }
    done.fetch_or(bit, std::memory_order_relaxed);
    return SLLM_OK;
}

template <typename T, int HD>
int append_hd(const sllm_kv8_layer* c, const sllm_kv8_rows* r, int sms, void* stream) {
    Append8Args a{view(c), r->k, r->v, reinterpret_cast<const long long*>(r->slot_map), (long long)r->k_stride, (long long)r->v_stride, (int)r->n_tok, 0};
    const size_t w = sizeof(T);
    a.wide = aligned(r->k, 16) && aligned(r->v, 16) && (r->k_stride * w) % 16 == 0 && (r->v_stride * w) % 16 == 0;
    const unsigned windows = (r->n_tok + kAppendWindow - 1) / kAppendWindow;
    // A window has between 1 run (a prompt) and 16 (a decode step), 2 kv_heads units each.  Short lists get a warp for
    // every unit there could be; long ones one for each unit of a prompt's window.
    const unsigned teams = kAppendWarps / (HD / 128 + 1), most = (2 * c->kv_heads * kAppendWindow + teams - 1) / teams, least = (2 * c->kv_heads + teams - 1) / teams;
    const unsigned y = std::min(most, std::max(least, (unsigned)(sms * 16) / windows));
    return launch("sllm_k_kv8_append", k_kv8_append<T, HD>, dim3(windows, y), kAppendWarps * 32, 0, stream, a);
}
template <typename T>
int append_t(const sllm_kv8_layer* c, const sllm_kv8_rows* r, int sms, void* stream) {
    switch (c->head_dim) {
        case 16: return append_hd<T, 16>(c, r, sms, stream);
        case 32: return append_hd<T, 32>(c, r, sms, stream);
        case 64: return append_hd<T, 64>(c, r, sms, stream);
        default: return append_hd<T, 128>(c, r, sms, stream);
    }
}

template <typename T, int HD>
int read_hd(const sllm_kv8_layer* c, const Read8Args& a, void* stream) {
    constexpr int rows = kReadThreads / (HD / 8) * 4;
    return launch("sllm_k_kv8_read", k_kv8_read<T, HD>, dim3((a.n_tok + rows - 1) / rows, 2 * c->kv_heads), kReadThreads, 0, stream, a);
}
template <typename T>
int read_t(const sllm_kv8_layer* c, const Read8Args& a, void* stream) {
    switch (c->head_dim) {
        case 16: return read_hd<T, 16>(c, a, stream);
        case 32: return read_hd<T, 32>(c, a, stream);
        case 64: return read_hd<T, 64>(c, a, stream);
        default: return read_hd<T, 128>(c, a, stream);
    }
}

int check_rows(const char* what, const sllm_kv8_layer* c, const sllm_kv8_rows* r, int* dev, int* sms) {
    if (int rc = check_layer(what, c)) return rc;
    if (!r || !r->k || !r->v || !r->slot_map) return bad(what, "null pointer");
    if (r->dtype != SLLM_ROWS_BF16 && r->dtype != SLLM_ROWS_F32) return bad(what, "dtype must be SLLM_ROWS_BF16 or SLLM_ROWS_F32");
    if (r->n_tok > 0x40000000u) return bad(what, "too many rows");
    const uint64_t row = (uint64_t)c->kv_heads * c->head_dim;
    if (r->k_stride < row || r->v_stride < row || r->k_stride >> 40 || r->v_stride >> 40) return bad(what, "a row stride is shorter than kv_heads * head_dim, or absurd");
    const size_t w = r->dtype == SLLM_ROWS_BF16 ? 2 : 4;
    if (!aligned(r->k, w) || !aligned(r->v, w) || !aligned(r->slot_map, 8)) return bad(what, "misaligned pointer");
    if (int rc = current_device(what, dev, sms)) return rc;
    return check_memory(what, *dev, {c->pages, c->scales, r->k, r->v, r->slot_map});
}

// ---- attention: which form, how the work is cut -----------------------------------------------------------------
struct Plan { Attn8Args a; unsigned tiles; bool tc; };

Plan plan_attn(const sllm_kv8_layer* c, const sllm_kv8_attn* s, int sms) {
    Plan p{};
    Attn8Args& a = p.a;
    a.c = view(c);
    a.q = s->q; a.out = s->out; a.q_stride = (long long)s->q_stride; a.out_stride = (long long)s->out_stride;
    a.table = s->table; a.tok_seq = s->tok_seq; a.tok_pos = s->tok_pos;
    a.cu_tok = s->max_new == 1 ? nullptr : s->cu_tok;
    a.n_tok = (int)s->n_tok; a.n_seq = (int)s->n_seq; a.width = (int)s->table_width; a.n_heads = (int)s->n_heads;
    a.group = (int)(s->n_heads / c->kv_heads);
    a.head_tiles = (a.group + kA8Rows - 1) / kA8Rows;
    a.rows_heads = (a.group + a.head_tiles - 1) / a.head_tiles;
    a.rows_toks = a.cu_tok ? kA8Rows / a.rows_heads : 1;
    p.tiles = a.cu_tok ? s->n_tok / a.rows_toks + s->n_seq : s->n_tok;
    const size_t w = s->dtype == SLLM_ROWS_BF16 ? 2 : 4;
    a.wide = aligned(s->q, 16) && aligned(s->out, 16) && (s->q_stride * w) % 16 == 0 && (s->out_stride * w) % 16 == 0;
    a.scale = s->scale != 0.f ? s->scale : 1.0f / std::sqrt((float)c->head_dim);
    a.status = s->status;
    // bf16 rows of runs of many (tokens x heads of a group) take the tensor-core form, whose tiles of 128 rows cost the same whatever
    // part of them is filled.  Ten heads of 64, us there and in the general form: 64 sequences of 1 to 64 new tokens (32 rows on
    // average) 87 and 71, 16 of 16 to 80 (48 rows) 30 and 43, 4 of 200 17 and 37.
    p.tc = a.cu_tok && s->dtype == SLLM_ROWS_BF16 && c->head_dim >= 64 && a.group <= kT8Rows && (uint64_t)s->n_tok * a.group >= 40ull * s->n_seq &&
           s->n_tok / (kT8Rows / a.group) + (uint64_t)s->n_seq <= 65535;
    const long long most = (long long)s->table_width * kPage, len = s->max_len ? std::min<long long>(s->max_len, most) : most;
    if (p.tc) {
        // Two tiles of query rows per block share the widening of K and V, which pays at head_dim 128 (in small grids too: 300 tokens of
        // 4 sequences 60 us either way, 2000 of one 64 us against 74); at 64 one leaves two blocks to an SM, which hides a block's
        // beginning and end.
        const int nt = c->head_dim == 64 ? 1 : 2;
        a.rows_toks = nt * (kT8Rows / a.group);
        p.tiles = s->n_tok / a.rows_toks + s->n_seq;
        // Chunks, of at least 1024 keys, only where the blocks would not fill half the GPU: their states are fp32 rows in the workspace
        // (a step with 3100 tokens in three chunks 108 us, uncut 77).
        const long long base = (long long)p.tiles * c->kv_heads, slots = (nt == 1 ? 2ll : 1ll) * sms;
        const long long chunks = std::max(1ll, std::min(slots / base, len / 1024));
        a.chunk = (int)((len + chunks * kPage - 1) / (chunks * kPage)) * kPage;
        a.n_chunks = (int)std::max(1ll, (len + a.chunk - 1) / a.chunk);
        return p;
    }
    // Chunks of the keys until there are about two rounds of blocks, none shorter than a unit per warp nor longer than 4096 keys (of
    // rows of very different lengths; four documents of 60 to 131 thousand keys: 149 us without that, 132 with).  Few short rows are
    // cut into at most eight, which a cluster joins: 6.9 us for ten heads of 2048 keys, where sixteen chunks and a second kernel
    // take 7.6; with more blocks than two or three per SM the cluster's blocks wait for one another (16 sequences: 21 us, 14 without).
    const long long base = (long long)p.tiles * c->kv_heads * a.head_tiles;
    const long long want = 2ll * sms * (c->head_dim > 64 ? 3 : 4);
    constexpr long long least = kA8Warps * kA8Unit, longest = 4096;
    long long chunks = std::max((want + base - 1) / base, base < want ? (len + longest - 1) / longest : 1ll);
    chunks = std::max(1ll, std::min({chunks, (len + least - 1) / least, (long long)kA8MaxChunks}));
    const bool few = len <= 2 * least * kA8MaxCluster && base * std::min<long long>(chunks, kA8MaxCluster) <= 5ll * sms / 2;
    if (few) chunks = std::min<long long>(chunks, kA8MaxCluster);
    long long chunk = (len + chunks - 1) / chunks;
    chunk = (chunk + least - 1) / least * least;
    a.chunk = (int)chunk;
    a.n_chunks = (int)std::max(1ll, (len + chunk - 1) / chunk);
    a.cluster = few && a.n_chunks > 1;
    return p;
}
uint64_t plan_bytes(const Plan& p, uint32_t hd) {
    return p.a.n_chunks > 1 && !p.a.cluster ? (uint64_t)p.a.n_tok * p.a.n_heads * p.a.n_chunks * (hd + 2) * sizeof(float) : 0;
}

int check_attn(const char* what, const sllm_kv8_layer* c, const sllm_kv8_attn* a) {
    if (int rc = check_layer(what, c)) return rc;
    if (!a || !a->q || !a->out || !a->table || !a->tok_seq || !a->tok_pos) return bad(what, "null pointer");
    if (a->dtype != SLLM_ROWS_BF16 && a->dtype != SLLM_ROWS_F32) return bad(what, "dtype must be SLLM_ROWS_BF16 or SLLM_ROWS_F32");
    if (a->n_heads < 1 || a->n_heads % c->kv_heads != 0 || a->n_heads > 65535) return bad(what, "n_heads must be a multiple of kv_heads");
    if (a->n_seq < 1 || a->n_seq > 0x1000000u || a->n_tok > 0x1000000u) return bad(what, "n_seq must be 1..2^24, n_tok at most 2^24");
    if (a->table_width < 1 || a->table_width > 0x1000000u) return bad(what, "table_width must be 1..2^24");
    const uint64_t row = (uint64_t)a->n_heads * c->head_dim;
    if (a->q_stride < row || a->out_stride < row || a->q_stride >> 40 || a->out_stride >> 40) return bad(what, "a row stride is shorter than n_heads * head_dim, or absurd");
    const size_t w = a->dtype == SLLM_ROWS_BF16 ? 2 : 4;
    if (!aligned(a->q, w) || !aligned(a->out, w) || !aligned(a->table, 4) || !aligned(a->tok_seq, 4) || !aligned(a->tok_pos, 4) || !aligned(a->cu_tok, 4) || !aligned(a->status, 4))
        return bad(what, "misaligned pointer");
    if (!std::isfinite(a->scale)) return bad(what, "scale must be finite");
    if (a->n_tok) {
        const char *q0 = static_cast<const char*>(a->q), *q1 = q0 + ((a->n_tok - 1) * a->q_stride + row) * w;
        const char *o0 = static_cast<const char*>(a->out), *o1 = o0 + ((a->n_tok - 1) * a->out_stride + row) * w;
        if (q0 < o1 && o0 < q1) return bad(what, "q and out overlap");
    }
    return SLLM_OK;
}

template <typename T, int HD>
int join_chunks(const Attn8Args& a, void* stream) {
    return launch("sllm_k_attn_kv8", k_attn_kv8_join<T, HD>, dim3((unsigned)a.n_tok * a.n_heads), 128, 0, stream, a);
}
template <typename T, int HD, bool I8, bool CL>
int attn_form(const Plan& p, int dev, void* stream) {
    static std::atomic<uint64_t> done{0};
    const char* what = "sllm_k_attn_kv8";
    if (int rc = opt_in(what, k_attn_kv8<T, HD, I8, CL>, attn8_smem<HD>(), dev, done)) return rc;
    const Attn8Args& a = p.a;
    const uint64_t blocks = (uint64_t)p.tiles * a.c.H * a.head_tiles;
    if (blocks > 0x7fffffffu) return bad(what, "too many rows and heads for one call");
    const dim3 grid((unsigned)blocks, 1, a.n_chunks);
    if (int rc = launch_cluster(what, k_attn_kv8<T, HD, I8, CL>, grid, kA8Threads, attn8_smem<HD>(), stream, CL ? a.n_chunks : 1, a)) return rc;
    if (a.n_chunks == 1 || CL) return SLLM_OK;
    return join_chunks<T, HD>(a, stream);
}
template <typename T, int HD>
int attn_hd(const Plan& p, int dev, void* stream) {
    constexpr bool i8 = std::is_same<T, __nv_bfloat16>::value && HD >= 32;           // the integer form: bf16 rows
    return p.a.cluster ? attn_form<T, HD, i8, true>(p, dev, stream) : attn_form<T, HD, i8, false>(p, dev, stream);
}
template <int HD, int NT>
int attn_tc(const Plan& p, int dev, void* stream) {
    static std::atomic<uint64_t> done{0};
    const char* what = "sllm_k_attn_kv8";
    if (int rc = opt_in(what, k_attn_kv8_tc<HD, NT>, attn8_tc_smem<HD, NT>(), dev, done)) return rc;
    if (int rc = launch(what, k_attn_kv8_tc<HD, NT>, dim3(p.a.c.H, p.tiles, p.a.n_chunks), attn8_tc_threads<NT>(), attn8_tc_smem<HD, NT>(), stream, p.a)) return rc;
    return p.a.n_chunks == 1 ? SLLM_OK : join_chunks<__nv_bfloat16, HD>(p.a, stream);
}
template <typename T>
int attn_t(const Plan& p, uint32_t hd, int dev, void* stream) {
    switch (hd) {
        case 16: return attn_hd<T, 16>(p, dev, stream);
        case 32: return attn_hd<T, 32>(p, dev, stream);
        case 64: return attn_hd<T, 64>(p, dev, stream);
        default: return attn_hd<T, 128>(p, dev, stream);
    }
}

}  // namespace

extern "C" {

int sllm_k_block_tables(const sllm_block_tables* s, void* stream) {
    const char* what = "sllm_k_block_tables";
    if (!s || !s->len_before || !s->len_after || !s->table || !s->ring || !s->pool_in || !s->pool_out || !s->cu_tok || !s->tok_seq || !s->tok_pos || !s->slot_map)
        return bad(what, "null pointer");
    if (s->n_seq < 1 || s->n_seq > (uint32_t)kTablesMaxSeq) return bad(what, "n_seq must be 1..8192");
    if (s->table_width < 1 || s->table_width > 0x1000000u) return bad(what, "table_width must be 1..2^24");
    if (s->n_pages < 1 || s->n_pages > 0x7fffffffull) return bad(what, "n_pages must be 1..2^31 - 1");
    if (s->max_tok > 0x40000000u) return bad(what, "max_tok is too large");
    if (s->pool_in < s->pool_out + 4 && s->pool_out < s->pool_in + 4) return bad(what, "pool_in and pool_out overlap");
    if (!aligned(s->len_before, 4) || !aligned(s->len_after, 4) || !aligned(s->table, 4) || !aligned(s->ring, 4) || !aligned(s->pool_in, 8) || !aligned(s->pool_out, 8) ||
        !aligned(s->cu_tok, 4) || !aligned(s->tok_seq, 4) || !aligned(s->tok_pos, 4) || !aligned(s->slot_map, 8))
        return bad(what, "misaligned pointer");
    int dev, sms;
    if (int rc = current_device(what, &dev, &sms)) return rc;
    if (int rc = check_memory(what, dev, {s->len_before, s->len_after, s->table, s->ring, s->pool_in, s->pool_out, s->cu_tok, s->tok_seq, s->tok_pos, s->slot_map})) return rc;
    TablesArgs a{s->len_before, s->len_after, s->table, s->ring, reinterpret_cast<const long long*>(s->pool_in), reinterpret_cast<long long*>(s->pool_out), s->cu_tok,
                 s->tok_seq, s->tok_pos, reinterpret_cast<long long*>(s->slot_map), (long long)s->n_pages, (int)s->n_seq, (int)s->table_width, (int)s->max_tok};
    static std::atomic<uint64_t> done{0};
    if (int rc = opt_in(what, k_block_tables, 3 * (kTablesMaxSeq + 1) * sizeof(int), dev, done)) return rc;
    // Every block sums over all sequences: small blocks are quicker at few of them (24 sequences, 3100 entries: 2.7 us against 5.8), but a
    // thread of theirs has many.
    const int block = s->n_seq <= 1024 ? 256 : 1024;
    const unsigned grid = std::max(1u, std::min((unsigned)sms, (s->max_tok + block - 1) / block));
    return launch(what, k_block_tables, dim3(grid), block, 3 * (size_t)(s->n_seq + 1) * sizeof(int), stream, a);
}

int sllm_k_kv8_append(const sllm_kv8_layer* c, const sllm_kv8_rows* r, void* stream) {
    int dev, sms;
    if (int rc = check_rows("sllm_k_kv8_append", c, r, &dev, &sms)) return rc;
    if (r->n_tok == 0) return SLLM_OK;
    return r->dtype == SLLM_ROWS_F32 ? append_t<float>(c, r, sms, stream) : append_t<__nv_bfloat16>(c, r, sms, stream);
}

int sllm_k_kv8_read(const sllm_kv8_layer* c, const sllm_kv8_rows* r, void* stream) {
    const char* what = "sllm_k_kv8_read";
    int dev, sms;
    if (int rc = check_rows(what, c, r, &dev, &sms)) return rc;
    if (r->n_tok == 0) return SLLM_OK;
    const size_t w = r->dtype == SLLM_ROWS_BF16 ? 2 : 4;
    Read8Args a{view(c), const_cast<void*>(r->k), const_cast<void*>(r->v), reinterpret_cast<const long long*>(r->slot_map), (long long)r->k_stride, (long long)r->v_stride,
                (int)r->n_tok, 0};
    a.wide = aligned(r->k, 16) && aligned(r->v, 16) && (r->k_stride * w) % 16 == 0 && (r->v_stride * w) % 16 == 0;
    return r->dtype == SLLM_ROWS_F32 ? read_t<float>(c, a, stream) : read_t<__nv_bfloat16>(c, a, stream);
}

int sllm_k_attn_kv8_workspace(const sllm_kv8_layer* c, const sllm_kv8_attn* s, uint64_t* bytes) {
    const char* what = "sllm_k_attn_kv8_workspace";
    if (!bytes) return bad(what, "null pointer");
    if (int rc = check_attn(what, c, s)) return rc;
    int dev, sms;
    if (int rc = current_device(what, &dev, &sms)) return rc;
    *bytes = s->n_tok ? plan_bytes(plan_attn(c, s, sms), c->head_dim) : 0;
    return SLLM_OK;
}

int sllm_k_attn_kv8(const sllm_kv8_layer* c, const sllm_kv8_attn* s, void* workspace, uint64_t workspace_bytes, void* stream) {
    const char* what = "sllm_k_attn_kv8";
    if (int rc = check_attn(what, c, s)) return rc;
    int dev, sms;
    if (int rc = current_device(what, &dev, &sms)) return rc;
    if (int rc = check_memory(what, dev, {c->pages, c->scales, s->q, s->out, s->table, s->tok_seq, s->tok_pos, s->cu_tok, s->status, workspace})) return rc;
    if (s->n_tok == 0) return SLLM_OK;
    Plan p = plan_attn(c, s, sms);
    if ((uint64_t)s->n_tok * s->n_heads > 0x7fffffffu) return bad(what, "too many rows and heads for one call");
    const uint64_t need = plan_bytes(p, c->head_dim);
    if (need) {
        if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
            return bad(what, "the workspace is missing, misaligned (16 bytes) or smaller than sllm_k_attn_kv8_workspace says");
        p.a.part = static_cast<float*>(workspace);
        p.a.part_ml = p.a.part + (size_t)p.a.n_tok * p.a.n_heads * p.a.n_chunks * c->head_dim;
    }
    if (p.tc) return c->head_dim == 64 ? attn_tc<64, 1>(p, dev, stream) : attn_tc<128, 2>(p, dev, stream);
    return s->dtype == SLLM_ROWS_F32 ? attn_t<float>(p, c->head_dim, dev, stream) : attn_t<__nv_bfloat16>(p, c->head_dim, dev, stream);
}

}  // extern "C"
