// Attention over the 8-bit paged cache (kv8.cuh) for few query rows per sequence: decode, drafts, grouped heads, and the
// general form for every type and size.
//
//   o = sum_j p_j vs_b(j) V_j / sum_j p_j,   p_j = exp(scale ks_b(j) (q . K_j) - m),   j <= position of the row
//
// with K_j, V_j the stored integers and ks, vs the scales of their blocks of 16 positions.  Only a block's scale touches an
// integer product, so the products run on the integers themselves: mma.sync with eight query rows (tokens x heads that share
// a kv head) as its rows 0..7, and what the 8 or 11 bits of an operand leave out of them as its rows 8..15, so that both parts
// come out in one thread and are added there, at no more matrix instructions than one row costs.  q is first divided by a power
// of two so that its largest value is in [0.5, 1).  The products with V are of one unit of 32 keys at a time: its weights p vs are taken
// relative to their own largest, and the unit's sum is added, with that factor, to an fp32 accumulator relative to m.  So the
// precision of a weight is that of its unit: neither the loudest value of the cache, nor a strong key (an attention sink) elsewhere
// in it, takes bits from what many small weights add up to.  Two forms:
//   bf16 rows (I8): m16n8k32 on int8, the cache's bytes as they are.  q and p vs become two base-256 digits, 16 bits in all: q, multiplied
//     by a power of two, exactly down to 2^-7 of the row's largest value (2^-6 where its bits are all ones) and to 2^-15 of that below, p vs to
//     2^-16 of the unit's largest (the output is rounded to 2^-9).  Products and a unit's sums are exact, in 32-bit integers.
//   fp32 rows: m16n8k16 on fp16, in which the integers are exact, q and p vs split into a high and a low fp16 part, 22 bits (p vs to 2^-39
//     of the unit's largest at least), fp32 sums: fp32 accuracy.  A byte costs 1.25-1.5 instructions on its way there (xor the sign, byte-permute under 0x64
//     = 1024 + x, subtract), where I8 spends none on K and half of one on V, to bring four keys of a dim into one register.
//
// The kernel is to be bound by HBM: 2 head_dim bytes per cached position and kv head.  A block of threads takes one (row
// tile, kv head, chunk of the keys); each of its four warps takes every fourth unit of 32 keys, through bulk copies of its own,
// two units ahead, and has its own running state; the states are joined once.  Keys are cut into chunks when there are few
// rows: of a few short rows at most eight, the blocks of a cluster, which join their states through one another's shared memory;
// otherwise the states go to the workspace, and a second, small kernel joins them.
// Measured (of the 6460 GB/s of a copy; the kernel repeated in a graph, and with caches that other passes have left cold): 512 sequences of
// 256 to 2047 positions, ten heads of 64, 124 and 142 us = 6.2 and 5.4 TB/s; four of 60 to 131
// thousand, 8 kv heads of 128 with four query heads each, 138 and 147 us = 5.7 and 5.4 TB/s; one of 2048, ten heads, 7 us, which is latency: the
// lists, the table, the pages, the join.  With fp16 products for bf16 rows too the first took 178 us, bound by instruction issue.  A running
// reference for all units' weights and 32-bit integer accumulators, which a strong key leaves too few bits, took 127 us: 96
// registers and not 80, five blocks per SM and not six.
#pragma once
#include <cuda_fp16.h>

#include <type_traits>

#include "attn_stream.cuh"
#include "kv8.cuh"

namespace sllm {

constexpr int kA8Warps = 4;
constexpr int kA8Threads = kA8Warps * 32;
constexpr int kA8Stages = 2;           // units in flight per warp: more would cost a block per SM (512 sequences: 3 stages 139 us, 2 stages 128 us)
constexpr int kA8Unit = 32;            // keys per step of a warp: two blocks of 16
constexpr int kA8Rows = 8;             // query rows of a tile

struct Attn8Args {
    Kv8View c;
    const void* q; void* out;          // [n_tok][n_heads][hd], rows q_stride / out_stride elements apart
    long long q_stride, out_stride;
    const int* table;                  // [n_seq][width]
    const int* tok_seq; const int* tok_pos;    // [n_tok]
    const int* cu_tok;                 // [n_seq + 1], or null: every token is a tile of its own
    int n_tok, n_seq, width, n_heads, group;   // group = n_heads / kv heads
    int rows_heads;                    // heads of a tile (<= 8), head_tiles tiles cover a group
    int head_tiles;
    int rows_toks;                     // tokens of a tile
    int chunk;                         // keys per chunk, a multiple of 64
    int n_chunks;
    int wide;                          // q and out rows are 16-byte aligned
    float scale;
    int cluster;                       // they are a cluster's blocks
    float* part;                       // n_chunks > 1 without a cluster: [n_tok][n_heads][n_chunks][hd] sums, then [..][2] (m in log2 units, l)
    float* part_ml;
    int* status;                       // optional
};

template <int HD> __host__ __device__ constexpr size_t attn8_smem() {
    // per warp and stage: K rows, V rows, eight scales (64 bytes reserved)
    return (size_t)kA8Warps * kA8Stages * (2 * kA8Unit * HD + 64);
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16832(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four values times a factor, at most 32639 and rounded, as two base-256 digits each: the high ones in [-127, 127], the low ones in
// [-128, 127].  (Weights, in [0, 1], times 32512.)  The sum with 1.5 * 2^23 + 128 leaves the integer, 128 up, in the low bits: its second byte is the high digit and
// its first, sign flipped, the low one.
constexpr float kDigits = 32512.f;
constexpr float kSplitTop = 16384.f;   // what a unit's largest weight of the fp16 form is brought to: its parts are then good to 2^-39 of it
__device__ __forceinline__ uint32_t digit_bits(float x, float f) { return __float_as_uint(fmaf(x, f, 12583040.f)); }
__device__ __forceinline__ void digits4(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3, uint32_t& hi, uint32_t& lo) {
    const uint32_t a = __byte_perm(x0, x1, 0x5140), b = __byte_perm(x2, x3, 0x5140);      // low, low, high, high
    lo = __byte_perm(a, b, 0x5410) ^ 0x80808080u;
    hi = __byte_perm(a, b, 0x7632);
}
// bytes 0, 1 (or 2, 3) of four excess-128 bytes as two halves: 0x64xx is 1024 + xx, minus 1152 leaves the signed value
__device__ __forceinline__ uint32_t halves(uint32_t w, uint32_t sel) {
    const uint32_t x = __byte_perm(w, 0x64646464u, sel);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// high and low fp16 parts of two floats
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    const float2 f = __half22float2(h);
    lo = pack_half(a - f.x, b - f.y);
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// smallest power of two >= x, for 0 <= x < infinity (0 for 0)
__device__ __forceinline__ float pow2_above(float x) {
    const uint32_t u = __float_as_uint(x);
    return __uint_as_float((u + 0x007fffffu) & 0x7f800000u);
}
// the row tile of a block: tokens [t0, t0 + n) of one sequence (n = 0: nothing to do); cu: a.cu_tok, or a copy of it
__device__ __forceinline__ int attn8_tile(const Attn8Args& a, const int* cu, int tile, int& t0, int& seq) {
    if (!cu) {
        t0 = tile;
        seq = a.tok_seq[tile];
        return seq >= 0 && seq < a.n_seq ? 1 : 0;
    }
    // sequence i gets tile numbers from cu[i] / rows_toks + i on: at least as many as it needs, and found by a binary search
    int lo = 0, hi = a.n_seq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] / a.rows_toks + mid <= tile) lo = mid; else hi = mid;
    }
    const int first = cu[lo];
    const int end = min(cu[lo + 1], a.n_tok);
    t0 = first + (tile - first / a.rows_toks - lo) * a.rows_toks;
    seq = lo;
    return first >= 0 && t0 >= 0 ? min(a.rows_toks, end - t0) : 0;
}
constexpr int kA8MaxCluster = 8;       // blocks of a cluster: what every GPU grants
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the float at the same place of shared memory in the cluster's block `rank`
__device__ __forceinline__ float peer_f32(const float* p, int rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(as_smem(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float4 peer_f32x4(const float* p, int rank) {
    uint32_t at;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(as_smem(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}
// weight of a part with maximum mp and sum lp in a whole with maximum m: a part whose scores are all NaN has no maximum, but its sum says so
__device__ __forceinline__ float part_weight(float mp, float lp, float m) { return mp == -INFINITY ? (lp == 0.f ? 0.f : 1.f) : exp2_fast(mp - m); }
// chunks of a tile whose last row stands at `last`
__device__ __forceinline__ int attn8_chunks(const Attn8Args& a, int last) { return (int)min(((long long)last + a.chunk) / a.chunk, (long long)a.n_chunks); }

// CL: the chunks of a tile are a cluster's blocks (a form of its own: it costs registers, and with them blocks per SM)
template <typename T, int HD, bool I8, bool CL>
__global__ void __launch_bounds__(kA8Threads) k_attn_kv8(const Attn8Args a) {
    static_assert(!I8 || HD >= 32, "a k step of the integer products has 32 dims");
    constexpr int KS = HD / (I8 ? 32 : 16);      // k steps of the score product
    constexpr int KB = HD / 4;                   // bytes of a key row per lane
    constexpr int VB = HD / 8;                   // bytes of a value row per lane = column tiles of the output
    constexpr uint32_t RUN = kA8Unit * HD;       // bytes of a unit's K (or V) rows
    constexpr uint32_t STAGE = 2 * RUN + 64;
    constexpr int ST = kA8Stages;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long bars[kA8Warps][ST];
    __shared__ float s_m[kA8Warps][kA8Rows], s_l[kA8Warps][kA8Rows];
    __shared__ float s_cm[CL ? kA8Rows : 1], s_cl[CL ? kA8Rows : 1];
    __shared__ __align__(16) float s_co[CL ? kA8Rows : 1][CL ? HD : 4];      // the block's joined state, for the cluster
    __shared__ int s_ok;
    __shared__ unsigned s_live;                  // bit 4 r: row r is somebody's

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    if (tid == 0) {
        for (int w = 0; w < kA8Warps; ++w)
            for (int s = 0; s < ST; ++s) bar_init(as_smem(&bars[w][s]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        s_ok = 1;
    }
    pdl_launch_dependents();
    pdl_wait();
    // heads follow on one another: the blocks that run side by side read the same pages, whose heads lie next to each other
    const int per_tile = a.c.H * a.head_tiles, tile = blockIdx.x / per_tile, in_tile = blockIdx.x % per_tile;
    int t0, seq;
    const int n = attn8_tile(a, a.cu_tok, tile, t0, seq);
    if (n <= 0) return;
    const int head = in_tile / a.head_tiles, ht = in_tile % a.head_tiles;
    const int chunk = blockIdx.z;
    // this lane's row
    const int r_tok = g / a.rows_heads, r_head = ht * a.rows_heads + g % a.rows_heads;
    // an entry in a sequence's run that does not name it is skipped (without cu_tok the entry has named its sequence); both loads at once
    int who = -1, at = -1;
    if (r_tok < n && r_head < a.group) { at = a.tok_pos[t0 + r_tok]; who = a.cu_tok ? a.tok_seq[t0 + r_tok] : seq; }
    const bool row_ok = who == seq;
    const unsigned rows = __ballot_sync(0xffffffffu, row_ok);
    if (tid == 0) s_live = rows;
    const int pos = row_ok ? max(min(at, a.width * kPage - 1), -1) : -1;      // width * 64 is at most 2^30; not below -1: no difference wraps
    int last = pos;
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
    const int k0 = chunk * a.chunk;              // n_chunks * chunk may pass what this tile has; the last chunk takes all that is left
    const int keys = chunk == a.n_chunks - 1 ? last + 1 - k0 : min(last + 1 - k0, a.chunk);
    if (keys <= 0 && chunk > 0 && !CL) return;          // chunk 0 writes the rows that attend nothing
    __syncthreads();                             // barriers are initialised

    // the query rows as the A operand: reg 0, 2: this row's high parts; 1, 3: its low parts
    uint32_t qa[KS][4];
    float row_f;
    {
        float x[KB];
        const T* src = static_cast<const T*>(a.q) + (long long)(t0 + (row_ok ? r_tok : 0)) * a.q_stride + (head * a.group + (row_ok ? r_head : 0)) * HD + t * KB;
        if constexpr (KB >= 8) {
#pragma unroll
            for (int i = 0; i < KB; i += 8) load8(src + i, a.wide, x + i);
        } else {
#pragma unroll
            for (int i = 0; i < KB; ++i) x[i] = to_float(src[i]);
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < KB; ++i) top = fmaxf(top, fabsf(x[i]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // f = 2^(h - e) with top in [2^(e-1), 2^e), and its inverse: with h both are normal numbers up to the largest e, and the
        // low fp16 parts good to 2^-39 of the largest value.  Digits are of q 2^(15 - e): a bf16 top whose bits are all ones, which would
        // pass 127 * 256 + 127 there, counts as the next power of two.
        const int e = min(max((int)((__float_as_uint(top) + (I8 ? 0x10000u : 0u)) >> 23) - 126, -125), 129), h = e > -100 ? 14 : 0;
        const float f = top > 0.f ? __uint_as_float((uint32_t)(127 + h - e) << 23) : 1.f;
        row_f = (top > 0.f ? __uint_as_float((uint32_t)(127 + e - h) << 23) : 1.f) * a.scale * 1.4426950408889634f;
        if constexpr (I8) {
            // digits know no infinity and no NaN: the row's factor carries them
            float odd = 0.f;
#pragma unroll
            for (int i = 0; i < KB; ++i) odd = fmaf(x[i], 0.f, odd);
            odd += __shfl_xor_sync(0xffffffffu, odd, 1);
            odd += __shfl_xor_sync(0xffffffffu, odd, 2);
            row_f = row_f * (h ? 0.5f : 1.f / 32768.f) + odd;
            const float fd = h ? 2.f : 32768.f;          // f * fd may be no number of fp32: q is multiplied by one after the other
            const float f_ok = row_ok ? f : 0.f;
#pragma unroll
            for (int j = 0; j < KS; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float* y = x + 8 * j + 4 * i;
                    digits4(digit_bits(y[0] * f_ok, fd), digit_bits(y[1] * f_ok, fd), digit_bits(y[2] * f_ok, fd), digit_bits(y[3] * f_ok, fd), qa[j][2 * i], qa[j][2 * i + 1]);
                }
        } else
#pragma unroll
        for (int j = 0; j < KS; ++j) {
            if (!row_ok) { x[4 * j] = x[4 * j + 1] = x[4 * j + 2] = x[4 * j + 3] = 0.f; }
            split2(x[4 * j] * f, x[4 * j + 1] * f, qa[j][0], qa[j][1]);
            split2(x[4 * j + 2] * f, x[4 * j + 3] * f, qa[j][2], qa[j][3]);
        }
    }

    using Acc = typename std::conditional<I8, int, float>::type;
    float o[VB][2];
#pragma unroll
    for (int j = 0; j < VB; ++j) o[j][0] = o[j][1] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;

    const int n_units = keys > 0 ? (keys + kA8Unit - 1) / kA8Unit : 0;
    const int mine = n_units > warp ? (n_units - warp + kA8Warps - 1) / kA8Warps : 0;
    const int* table = a.table + (size_t)seq * a.width + k0 / kPage;
    unsigned char* my = smem_raw + (size_t)warp * ST * STAGE;
    // pages of 32 of this warp's units at a time, one per lane; -1 stands for a page outside the pool, whose keys do not count
    auto pages_of = [&](int i0) {
        const int u = (i0 + lane) * kA8Warps + warp;
        int p = -1;
        if (i0 + lane < mine) {
            p = table[u / (kPage / kA8Unit)];
            if (p < 0 || p >= a.c.n_pages) { p = -1; if (a.status) atomicExch(a.status, 1); }
        }
        return p;
    };
    int pid_iss = pages_of(0), pid_use = pid_iss;
    auto issue = [&](int i) {                    // the warp's unit i, by every lane (one of them copies)
        if ((i & 31) == 0 && i) pid_iss = pages_of(i);
        const int page = __shfl_sync(0xffffffffu, pid_iss, i & 31);
        if (page < 0 || lane != 0) return;
        const int s = i % ST, half_page = (i * kA8Warps + warp) % (kPage / kA8Unit);
        const uint32_t bar = as_smem(&bars[warp][s]), dst = as_smem(my + (size_t)s * STAGE);
        const long long run = ((long long)page * a.c.H + head) * 2;
        bar_expect(bar, 2 * RUN + 32);
        bulk_g2s(dst, a.c.pages + (run * kPage + half_page * kA8Unit) * HD, RUN, bar);
        bulk_g2s(dst + RUN, a.c.pages + ((run + 1) * kPage + half_page * kA8Unit) * HD, RUN, bar);
        bulk_g2s(dst + 2 * RUN, a.c.scales + run * kBlksPerPage, 32, bar);
    };
    for (int i = 0; i < ST && i < mine; ++i) issue(i);

    bool ok = true;
    uint32_t phase = 0;
    // row of key column g inside a group of 8: pairs of neighbours swap from the third pair on, so that the rows which one
    // load of V touches are not all even or all odd (rows are 64 bytes at head_dim 64: half the bank conflicts)
    const int key_of_g = g ^ ((g >> 2) & 1);
    for (int i = 0; i < mine; ++i) {
        if ((i & 31) == 0 && i) pid_use = pages_of(i);
        const int page = __shfl_sync(0xffffffffu, pid_use, i & 31);
        const int s = i % ST;
        if (page >= 0) {
            ok = bar_wait(as_smem(&bars[warp][s]), (phase >> s) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            phase ^= 1u << s;
            const unsigned char* sk = my + (size_t)s * STAGE;
            const unsigned char* sv = sk + RUN;
            const int unit = i * kA8Warps + warp;
            const float* scl = reinterpret_cast<const float*>(sk + 2 * RUN) + (unit % (kPage / kA8Unit)) * 2;
            const int kb = k0 + unit * kA8Unit;                  // first key of the unit
            float sc[4][2];
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
                Acc part[4] = {0, 0, 0, 0};
                uint32_t w[KB / 4];
                const unsigned char* row = sk + (nt * 8 + key_of_g) * HD + t * KB;
                if constexpr (KB >= 16) {
#pragma unroll
                    for (int x = 0; x < KB / 16; ++x) *reinterpret_cast<uint4*>(w + 4 * x) = *reinterpret_cast<const uint4*>(row + 16 * x);
                } else if constexpr (KB == 8) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(row);
                else w[0] = *reinterpret_cast<const uint32_t*>(row);
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    if constexpr (I8) mma16832(part, qa[j], w[2 * j], w[2 * j + 1]);
                    else {
                        const uint32_t b = w[j] ^ 0x80808080u;
                        mma16816(part, qa[j], halves(b, 0x4140), halves(b, 0x4342));
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) sc[nt][e] = I8 ? (float)((int)part[e] * 256 + (int)part[e + 2]) : (float)part[e] + (float)part[e + 2];
            }
            // scores in units of log2(e), masked by selection: what stands in a masked place is never used
            float mx = -INFINITY;
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
                const float f = scl[nt >> 1] * row_f;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int key = kb + nt * 8 + ((2 * t + e) ^ (t >> 1));
                    sc[nt][e] = key <= pos ? sc[nt][e] * f : -INFINITY;
                    mx = fmaxf(mx, sc[nt][e]);
                }
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(m_run, mx);
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            if (__any_sync(0xffffffffu, m_new != m_run)) {
                const float corr = exp2_fast(m_run - m_use);
                m_run = m_new;
                l_run *= corr;
#pragma unroll
                for (int j = 0; j < VB; ++j) { o[j][0] *= corr; o[j][1] *= corr; }
            }
            // the second block of a unit may lie behind the last position: its scale is another owner's then and does not count
            const float vs0 = scl[4], vs1 = kb + kBlk8 <= last ? scl[5] : 0.f;
            float top = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1])) + __log2f(vs0), fmaxf(fmaxf(sc[2][0], sc[2][1]), fmaxf(sc[3][0], sc[3][1])) + __log2f(vs1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // The unit's weights are p times these, k times what they are relative to its largest p vs, 2^top; its sum counts unit_f times.
            // Within 2^-120: what is below that adds nothing to a number that fp32 holds.
            constexpr float k = I8 ? kDigits : kSplitTop;
            const float unit_top = exp2_fast(fminf(fmaxf(top - m_use, -120.f), 126.f)), r = rcp_fast(unit_top), unit_f = unit_top * (1.f / k);
            const float g0 = fminf(vs0 * r * k, 3e38f), g1 = fminf(vs1 * r * k, 3e38f);   // 0 for a scale of 0, and finite: a p of 0 stays 0
            // a scale that is not finite shows by way of the sum: digits carry none, and g does not either
            if (!(vs0 < INFINITY) && kb <= pos) l_run = __uint_as_float(0x7fffffffu);
            if (!(vs1 < INFINITY) && kb + kBlk8 <= pos) l_run = __uint_as_float(0x7fffffffu);
            auto add = [&](int j, const Acc (&c)[4]) {           // a unit's product of column tile j
#pragma unroll
                for (int e = 0; e < 2; ++e) o[j][e] = fmaf(I8 ? (float)((int)c[e] * 256 + (int)c[e + 2]) : (float)c[e] + (float)c[e + 2], unit_f, o[j][e]);
            };
            if constexpr (I8) {
                uint32_t pa[4], x[8];
#pragma unroll
                for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float p = exp2_fast(sc[nt][e] - m_use);
                        l_run += p;
                        x[2 * nt + e] = digit_bits(p, nt >> 1 ? g1 : g0);
                    }
                digits4(x[0], x[1], x[2], x[3], pa[0], pa[1]);
                digits4(x[4], x[5], x[6], x[7], pa[2], pa[3]);
                // V: eight keys' rows, (2t, 2t + 1) of each group of 8 as permuted above; four bytes of four rows are turned into four
                // keys of four dims
                constexpr int NW = VB / 4;
                const int e0 = (2 * t) ^ (t >> 1), e1 = (2 * t + 1) ^ (t >> 1);
                uint32_t v[8][NW];
#pragma unroll
                for (int y = 0; y < 8; ++y) {
                    const unsigned char* src = sv + ((y & 1 ? e1 : e0) + (y >> 1) * 8) * HD + g * VB;
                    if constexpr (NW == 4) *reinterpret_cast<uint4*>(v[y]) = *reinterpret_cast<const uint4*>(src);
                    else if constexpr (NW == 2) *reinterpret_cast<uint2*>(v[y]) = *reinterpret_cast<const uint2*>(src);
                    else v[y][0] = *reinterpret_cast<const uint32_t*>(src);
                }
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    uint32_t b[2][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t r0 = __byte_perm(v[4 * h][w], v[4 * h + 1][w], 0x5140), r1 = __byte_perm(v[4 * h][w], v[4 * h + 1][w], 0x7362);
                        const uint32_t r2 = __byte_perm(v[4 * h + 2][w], v[4 * h + 3][w], 0x5140), r3 = __byte_perm(v[4 * h + 2][w], v[4 * h + 3][w], 0x7362);
                        b[h][0] = __byte_perm(r0, r2, 0x5410); b[h][1] = __byte_perm(r0, r2, 0x7632);
                        b[h][2] = __byte_perm(r1, r3, 0x5410); b[h][3] = __byte_perm(r1, r3, 0x7632);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) { int c[4] = {0, 0, 0, 0}; mma16832(c, pa, b[0][k], b[1][k]); add(4 * w + k, c); }
                }
            } else {
                uint32_t pa[2][4];
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    float p[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int key = kb + h * 8 + ((2 * t + e) ^ (t >> 1));
                        p[e] = exp2_fast(sc[h][e] - m_use);
                        l_run += p[e];
                        p[e] = key <= pos ? p[e] * (h >> 1 ? g1 : g0) : 0.f;
                    }
                    split2(p[0], p[1], pa[h >> 1][2 * (h & 1)], pa[h >> 1][2 * (h & 1) + 1]);
                }
                // V rows of keys (2t, 2t + 1) and (2t + 8, 2t + 9) of each block, as permuted above
                constexpr int NW = (VB + 3) / 4, NB = VB < 4 ? VB : 4;               // head_dim 16: two bytes of each row
                const int e0 = (2 * t) ^ (t >> 1), e1 = (2 * t + 1) ^ (t >> 1);
                uint32_t v[8][NW];
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const unsigned char* src = sv + ((x & 1 ? e1 : e0) + (x >> 1) * 8) * HD + g * VB;
                    if constexpr (VB == 16) *reinterpret_cast<uint4*>(v[x]) = *reinterpret_cast<const uint4*>(src);
                    else if constexpr (VB == 8) *reinterpret_cast<uint2*>(v[x]) = *reinterpret_cast<const uint2*>(src);
                    else if constexpr (VB == 4) v[x][0] = *reinterpret_cast<const uint32_t*>(src);
                    else v[x][0] = *reinterpret_cast<const uint16_t*>(src);
                }
#pragma unroll
                for (int w = 0; w < NW; ++w)
#pragma unroll
                    for (int y = 0; y < NB; y += 2) {                    // two dims at a time
                        float c[2][4] = {};
#pragma unroll
                        for (int kk = 0; kk < 2; ++kk) {
                            const uint32_t a2 = __byte_perm(v[4 * kk][w], v[4 * kk + 1][w], y ? 0x7362 : 0x5140) ^ 0x80808080u;
                            const uint32_t b2 = __byte_perm(v[4 * kk + 2][w], v[4 * kk + 3][w], y ? 0x7362 : 0x5140) ^ 0x80808080u;
                            mma16816(c[0], pa[kk], halves(a2, 0x4140), halves(b2, 0x4140));
                            mma16816(c[1], pa[kk], halves(a2, 0x4342), halves(b2, 0x4342));
                        }
                        add(4 * w + y, c[0]);
                        add(4 * w + y + 1, c[1]);
                    }
            }
            __syncwarp();                                        // every lane is done with stage s
        }
        if (i + ST < mine) issue(i + ST);
    }
    if (!ok) { s_ok = 0; l_run = __uint_as_float(0x7fffffffu); if (a.status) atomicExch(a.status, 5); }      // the tile's rows become NaN
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
    if (t == 0) { s_m[warp][g] = m_run; s_l[warp][g] = l_run; }
    __syncthreads();                                             // every warp is done with its stages: their memory is used again
    if (!s_ok)                                                   // let copies in flight land before shared memory is used again and released
        for (int i = 0; i < 32; ++i) __nanosleep(16384);
    constexpr int OS = HD + 4;                                   // floats per row: rows start in different banks
    static_assert((size_t)kA8Warps * kA8Rows * OS * 4 <= attn8_smem<HD>(), "the joined states fit the stages");
    float* so = reinterpret_cast<float*>(smem_raw);
#pragma unroll
    for (int j = 0; j < VB; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e)                              // column 2t + e of column tile j is dim (2t + e) VB + j
            so[(warp * kA8Rows + g) * OS + (2 * t + e) * VB + j] = o[j][e];
    __syncthreads();
    // eight dims per thread at a time: the four states joined in the order of the warps
    for (int x = tid; x < kA8Rows * HD / 8; x += kA8Threads) {
        const int r = x / (HD / 8), d = (x % (HD / 8)) * 8;
        const int rt = r / a.rows_heads, rh = ht * a.rows_heads + r % a.rows_heads;
        if (!(s_live >> (4 * r) & 1)) continue;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kA8Warps; ++w) m = fmaxf(m, s_m[w][r]);
        float l = 0.f, f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kA8Warps; ++w) {
            const float wt = part_weight(s_m[w][r], s_l[w][r], m);
            if (wt == 0.f && s_l[w][r] == 0.f) continue;
            l += wt * s_l[w][r];
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] += wt * so[(w * kA8Rows + r) * OS + d + k];
        }
        const long long tok = t0 + rt;
        const int qh = head * a.group + rh;
        if constexpr (CL) {
            store8(&s_co[r][d], true, f);
            if (d == 0) { s_cm[r] = m; s_cl[r] = l; }
        } else if (attn8_chunks(a, last) <= 1) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] *= inv;
            store8(static_cast<T*>(a.out) + tok * a.out_stride + qh * HD + d, a.wide, f);
        } else {
            const long long pi = (tok * a.n_heads + qh) * a.n_chunks + chunk;
            store8(a.part + pi * HD + d, true, f);
            if (d == 0) { a.part_ml[pi * 2] = m; a.part_ml[pi * 2 + 1] = l; }
        }
    }
    if constexpr (CL) {
    // The blocks' states, in their order: each block joins its share of the tile's values.
    cluster_barrier();
    for (int x = chunk * kA8Threads + tid; x < kA8Rows * HD / 4; x += a.n_chunks * kA8Threads) {
        const int r = x / (HD / 4), d = (x % (HD / 4)) * 4;
        const int rt = r / a.rows_heads, rh = ht * a.rows_heads + r % a.rows_heads;
        if (!(s_live >> (4 * r) & 1)) continue;
        float mp[kA8MaxCluster], lp[kA8MaxCluster], m = -INFINITY;
        float4 v[kA8MaxCluster];
#pragma unroll
        for (int c = 0; c < kA8MaxCluster; ++c)
            if (c < a.n_chunks) { mp[c] = peer_f32(&s_cm[r], c); lp[c] = peer_f32(&s_cl[r], c); v[c] = peer_f32x4(&s_co[r][d], c); }
#pragma unroll
        for (int c = 0; c < kA8MaxCluster; ++c)
            if (c < a.n_chunks) m = fmaxf(m, mp[c]);
        float l = 0.f, f[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kA8MaxCluster; ++c)
            if (c < a.n_chunks) {
                const float wt = part_weight(mp[c], lp[c], m);
                if (wt == 0.f && lp[c] == 0.f) continue;
                l += wt * lp[c];
                f[0] += wt * v[c].x; f[1] += wt * v[c].y; f[2] += wt * v[c].z; f[3] += wt * v[c].w;
            }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        T* dst = static_cast<T*>(a.out) + (long long)(t0 + rt) * a.out_stride + (head * a.group + rh) * HD + d;
#pragma unroll
        for (int k = 0; k < 4; ++k) dst[k] = from_float<T>(f[k] * inv);
    }
    cluster_barrier();                                           // nobody's shared memory goes while it is read
    }
}

// Joins the chunks of each (token, head), in their order: one block each.  A row whose tile had one chunk is written already;
// a tile's chunks are those of its last row, so a row may have chunks in which it attends nothing (m = -inf, l = 0).
// Bound by latency: all maxima in one round trip, all partial sums in another.
constexpr int kA8MaxChunks = 1024;
template <typename T, int HD>
__global__ void __launch_bounds__(128) k_attn_kv8_join(const Attn8Args a) {
    constexpr int LANES = HD / 4, GROUPS = 128 / LANES;          // a thread has four dims of every GROUPS-th chunk
    __shared__ float s_w[kA8MaxChunks], s_red[2][4], s_o[GROUPS][HD];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    const long long x = blockIdx.x;
    const int tok = (int)(x / a.n_heads), qh = (int)(x % a.n_heads);
    const int seq = a.tok_seq[tok];
    if (seq < 0 || seq >= a.n_seq) return;
    int first = tok, last = tok;                                 // the tile's tokens
    if (a.cu_tok) {
        const int c0 = a.cu_tok[seq], end = min(a.cu_tok[seq + 1], a.n_tok);
        if (tok < c0 || tok >= end) return;                      // the lists contradict one another: no tile had this row
        first = c0 + (tok - c0) / a.rows_toks * a.rows_toks;
        last = min(first + a.rows_toks, end) - 1;
    }
    int lp = -1;
    for (int i = first + lane; i <= last; i += 32)               // every warp for itself
        if (a.tok_seq[i] == seq) lp = max(lp, a.tok_pos[i]);
    lp = __reduce_max_sync(0xffffffffu, lp);
    lp = (int)min((long long)lp, (long long)a.width * kPage - 1);
    const int chunks = attn8_chunks(a, lp);
    if (chunks <= 1) return;
    const long long p0 = x * a.n_chunks;
    float m = -INFINITY;
    for (int c = tid; c < chunks; c += 128) { const float mc = a.part_ml[(p0 + c) * 2]; s_w[c] = mc; m = fmaxf(m, mc); }
    m = warp_max(m);
    if (lane == 0) s_red[0][warp] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
    float l = 0.f;
    for (int c = tid; c < chunks; c += 128) {
        const float mc = s_w[c], lc = a.part_ml[(p0 + c) * 2 + 1];
        const float w = part_weight(mc, lc, m);
        s_w[c] = w;
        l += w == 0.f && lc == 0.f ? 0.f : w * lc;
    }
    l = warp_sum(l);
    if (lane == 0) s_red[1][warp] = l;
    __syncthreads();
    l = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
    const int group = tid / LANES, d = (tid % LANES) * 4;
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = group; c < chunks; c += GROUPS) {
        const float w = s_w[c];
        const float4 v = *reinterpret_cast<const float4*>(a.part + (p0 + c) * HD + d);
        f.x += w * v.x; f.y += w * v.y; f.z += w * v.z; f.w += w * v.w;
    }
    *reinterpret_cast<float4*>(&s_o[group][d]) = f;
    __syncthreads();
    if (tid < HD) {
        float o = 0.f;
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) o += s_o[k][tid];
        static_cast<T*>(a.out)[(long long)tok * a.out_stride + qh * HD + tid] = from_float<T>(l == 0.f ? 0.f : o / l);
    }
}

}  // namespace sllm
