// The 8-bit paged KV cache: block tables and slot maps built on the GPU, appending rows, reading rows back.
//
// One layer of the cache is two arrays that the caller owns:
//   pages   int8 [n_pages][kv_heads][2][64][head_dim]     which = 0: K, 1: V
//   scales  fp32 [n_pages][kv_heads][2][4]                one for each block of 16 positions, head, and K or V
// A stored integer q stands for q * scale.  K and V of one (page, head) are one contiguous run (8 KB at head_dim 64), and
// so are their eight scales (32 bytes, one DRAM sector): a reader of a head fetches whole sectors of what it needs.
// Blocks of 16 rather than whole pages of 64: a scale costs 4 bytes per 16 * head_dim values either way next to nothing
// (0.4 % at head_dim 64), one loud row disturbs 15 others and not 63, and a row that raises a scale rewrites at most 15.
//
// Integers and not e4m3: with the scale taken from the block's own largest value, a uniform step of amax / 127 has a third
// of e4m3's root-mean-square error on normal data, and every int8 is exact in fp16, so the matrix instructions that
// attend the cache add no rounding of their own.
#pragma once
#include "common.cuh"

namespace sllm {

constexpr int kBlk8 = 16;                        // positions that share a scale
constexpr int kBlksPerPage = kPage / kBlk8;

struct Kv8View {
    int8_t* pages;
    float* scales;
    long long n_pages;
    int H;                                       // kv heads
};

// ---- block tables and slot maps -----------------------------------------------------------------------------------
struct TablesArgs {
    const int* before;       // [n_seq] positions held
    const int* after;        // [n_seq] positions held after the step
    int* table;              // [n_seq][width]
    int* ring;               // [n_pages] free pages, first in first out
    const long long* pool_in;    // {head, free, -, -}
    long long* pool_out;         // {head, free, tokens, status}
    int* cu_tok;             // [n_seq + 1]
    int* tok_seq; int* tok_pos; long long* slot_map;     // [room]
    long long n_pages;
    int n_seq, width, room;
};

constexpr int kTablesMaxSeq = 8192;              // three prefix arrays of this length fit shared memory (96 KB)

// Prefix sums over the sequences (new tokens, pages to take, pages to give back), then one thread per list entry.
// Every block repeats the sums, which costs each of them two loads per sequence, and so needs no second launch and no
// wait on another block.  What makes the blocks independent is that pages are taken from the ring's front and given back
// behind its end: with free + given back <= n_pages (checked) the two ranges never meet, the counters go to another buffer
// than they came from, and a thread that needs a page id reads it from the ring or from an entry that no thread writes.
// Bound by latency: one round trip for the lengths, one for the page, one store: 2.4 us for one sequence, 9.7 us for 4096 with 64
// thousand new positions (1 MB).
__global__ void __launch_bounds__(1024) k_block_tables(const TablesArgs a) {
    extern __shared__ int s_pre[];               // [3][n_seq + 1]
    __shared__ long long s_warp[3][32];
    const int n = a.n_seq, nt = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int* s_tok = s_pre;
    int* s_take = s_pre + (n + 1);
    int* s_give = s_pre + 2 * (n + 1);

    pdl_wait();
    const long long head = a.pool_in[0], free_pages = a.pool_in[1];
    const int per = (n + nt - 1) / nt, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    const long long most = (long long)a.width * kPage;
    long long sum[3] = {0, 0, 0};
    int bad = head < 0 || head >= a.n_pages || free_pages < 0 || free_pages > a.n_pages;
    for (int i = i0; i < i1; ++i) {
        const int b = a.before[i], e = a.after[i];
        if (b < 0 || e < 0 || b > most || e > most) { bad = 1; break; }
        const int have = (int)(((long long)b + kPage - 1) / kPage), need = (int)(((long long)e + kPage - 1) / kPage);
        sum[0] += max(0, e - b); sum[1] += max(0, need - have); sum[2] += max(0, have - need);
    }
    bad = __syncthreads_or(bad);
    // exclusive sums over the threads: inside a warp, then over the warps' totals
    long long ex[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        long long v = sum[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const long long u = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += u; }
        if (lane == 31) s_warp[k][warp] = v;
        ex[k] = v - sum[k];
    }
    __syncthreads();
    long long total[3] = {0, 0, 0};
    for (int w = 0; w < nt / 32; ++w)
#pragma unroll
        for (int k = 0; k < 3; ++k) { const long long v = s_warp[k][w]; if (w < warp) ex[k] += v; total[k] += v; }
    bad = bad || free_pages + total[2] > a.n_pages;
    const bool full = total[1] > free_pages || total[0] > a.room;
    const bool ok = !bad && !full;               // the same in every block: all or nothing
    if (ok)
        for (int i = i0; i < i1; ++i) {
            const int b = a.before[i], e = a.after[i];
            const int have = (b + kPage - 1) / kPage, need = (e + kPage - 1) / kPage;
            s_tok[i] = (int)ex[0]; s_take[i] = (int)ex[1]; s_give[i] = (int)ex[2];
            ex[0] += max(0, e - b); ex[1] += max(0, need - have); ex[2] += max(0, have - need);
        }
    if (tid == 0) { s_tok[n] = ok ? (int)total[0] : 0; s_take[n] = (int)total[1]; s_give[n] = (int)total[2]; }
    __syncthreads();
    const int n_tok = ok ? (int)total[0] : 0;

    if (blockIdx.x == 0) {
        for (int i = tid; i <= n; i += nt) a.cu_tok[i] = ok ? s_tok[i] : 0;
        if (tid == 0) {
            long long h = head + (ok ? total[1] : 0);
            if (ok && h >= a.n_pages) h -= a.n_pages;
            a.pool_out[0] = h;
            a.pool_out[1] = ok ? free_pages - total[1] + total[2] : free_pages;
            a.pool_out[2] = n_tok;
            a.pool_out[3] = ok ? 0 : (bad ? 1 : 4);              // SLLM_ERR_INVALID, SLLM_ERR_CAPACITY
        }
    }
    for (long long t = (long long)blockIdx.x * nt + tid; t < a.room; t += (long long)gridDim.x * nt) {
        int seq = -1, pos = -1;
        long long slot = -1;
        if (t < n_tok) {
            int lo = 0, hi = n;                                  // the last sequence that starts at or before t: it is not empty
            while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (s_tok[mid] <= t) lo = mid; else hi = mid; }
            seq = lo;
            const int b = a.before[seq];
            pos = b + (int)(t - s_tok[seq]);
            const int have = (b + kPage - 1) / kPage, pg = pos / kPage;
            int* entry = a.table + (size_t)seq * a.width + pg;
            int page;
            if (pg < have) page = *entry;
            else {
                long long r = head + s_take[seq] + (pg - have);
                if (r >= a.n_pages) r -= a.n_pages;
                page = a.ring[r];
                if (pos % kPage == 0) *entry = page;             // a new page's first position is always among the new ones
            }
            slot = (long long)page * kPage + pos % kPage;
        }
        a.tok_seq[t] = seq; a.tok_pos[t] = pos; a.slot_map[t] = slot;
    }
    if (ok && total[2] > 0)                                      // pages given back: a warp per sequence
        for (long long i = (long long)blockIdx.x * (nt / 32) + warp; i < n; i += (long long)gridDim.x * (nt / 32)) {
            const int give = s_give[i + 1] - s_give[i];
            const int need = (a.after[i] + kPage - 1) / kPage;
            for (int k = lane; k < give; k += 32) {
                long long r = head + free_pages + s_give[i] + k;
                if (r >= a.n_pages) r -= a.n_pages;
                if (r >= a.n_pages) r -= a.n_pages;
                a.ring[r] = a.table[(size_t)i * a.width + need + k];
            }
        }
}

// ---- rows of the caller's tensors ------------------------------------------------------------------------------------
// eight consecutive elements as floats; `wide`: base and row stride are multiples of 16 bytes
__device__ __forceinline__ void load8(const float* p, bool wide, float* f) {
    if (wide) {
        const float4 x = reinterpret_cast<const float4*>(p)[0], y = reinterpret_cast<const float4*>(p)[1];
        f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w; f[4] = y.x; f[5] = y.y; f[6] = y.z; f[7] = y.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = p[i];
    }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, bool wide, float* f) {
    if (wide) unpack16<__nv_bfloat16>(*reinterpret_cast<const uint4*>(p), f);
    else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __bfloat162float(p[i]);
    }
}
__device__ __forceinline__ void store8(float* p, bool wide, const float* f) {
    if (wide) {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = f[i];
    }
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, bool wide, const float* f) {
    if (wide) {
        uint4 v;
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) { const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&b); }
        *reinterpret_cast<uint4*>(p) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __float2bfloat16_rn(f[i]);
    }
}

// Eight values' rint(x / s), ties to even, as if the quotients were exact, as bytes.  x * (1 / s) rounded to an integer (by the
// addition of 1.5 * 2^23, which costs no conversion) is within one of it; the remainder x - q s is exact in one fma (|q| <= 127, and it is
// at most about s / 2, so its bits fit) and settles the rest, which is looked at only where it reaches s / 2.
__device__ __forceinline__ uint2 quant8(const float* x, float s, float inv) {
    constexpr float kBias = 12582912.f;
    uint32_t b[8];
    float r[8], worst = 0.f;
    const float half = 0.5f * s;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float y = fmaf(x[j], inv, kBias), q = y - kBias;
        b[j] = __float_as_uint(y);
        r[j] = fmaf(-q, s, x[j]);
        worst = fmaxf(worst, fabsf(r[j]));
    }
    if (worst >= half) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (r[j] > half || (r[j] == half && (b[j] & 1))) b[j] += 1;
            else if (r[j] < -half || (r[j] == -half && (b[j] & 1))) b[j] -= 1;
        }
    }
    const uint32_t b01 = __byte_perm(b[0], b[1], 0x0040), b23 = __byte_perm(b[2], b[3], 0x0040), b45 = __byte_perm(b[4], b[5], 0x0040), b67 = __byte_perm(b[6], b[7], 0x0040);
    return make_uint2(__byte_perm(b01, b23, 0x5410), __byte_perm(b45, b67, 0x5410));
}

// ---- append -------------------------------------------------------------------------------------------------------
struct Append8Args {
    Kv8View c;
    const void* k; const void* v;      // [n_tok][H][hd], rows k_stride / v_stride elements apart
    const long long* slot_map;         // [n_tok]; < 0 (or behind the pool): the row is skipped
    long long k_stride, v_stride;
    int n_tok, wide;
};

constexpr int kAppendWarps = 8;
constexpr int kAppendWindow = 16;      // list entries whose leaders one block handles

// A run: consecutive list entries whose slots follow on one another inside one block of 16 positions; its first entry
// leads it.  One warp takes one (run, head, K or V):
//   s = max(s_old, max|x| / 127)      s_old: the block's scale, 0 when the run starts the block
//   rows of the run: rint(x / s);  rows before it in the block, if s grew: rint(q s_old / s), in 64 bits
// A value that is not finite makes the scale NaN, and with it all that the block stands for: it shows in what attends
// it, and goes when the block is started anew.  The smallest scale of a block with anything in it is 2^-126, so that 1 / s
// is finite.
// A block of threads takes the leaders among 16 list entries (31 slots say where their runs end).  The rows are read once and
// kept in registers between the maximum and the rounding; at head_dim 128 two warps share a block of 16 rows, and registers are
// held to 80, so that three blocks of threads and not two fit an SM.  Bound by the bytes of long lists and the round trips to them, by latency in short ones:
// 2.5 us for 64 rows of ten heads of 64, 14.6 us for 7.4 thousand (28 MB; 17.5 with two blocks per SM), 20 us for eight thousand fp32 rows of eight heads of 128 (82 MB,
// 4.1 TB/s; 42 us with one warp per block and conversion instructions).
template <typename T, int HD>
__global__ void __launch_bounds__(kAppendWarps * 32, 3) k_kv8_append(const Append8Args a) {
    constexpr int VPR = HD / 8;                         // vectors of 8 per row
    constexpr int W = HD / 128 + 1, TEAM = W * 32;      // warps, threads of a unit
    constexpr int VPL = (kBlk8 * VPR + TEAM - 1) / TEAM;        // vectors per thread and unit
    __shared__ unsigned s_top[2][kAppendWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, team = warp / W, member = threadIdx.x % TEAM;
    const int t0 = blockIdx.x * kAppendWindow;
    pdl_wait();
    // lane l: slot of entry t0 - 1 + l
    const int te = t0 - 1 + lane;
    long long slot = -2;
    if (te >= 0 && te < a.n_tok) {
        slot = a.slot_map[te];
        if (slot < 0 || slot >= a.c.n_pages * kPage) slot = -2;
    }
    const long long prev = __shfl_up_sync(0xffffffffu, slot, 1);
    const bool live = slot >= 0;
    const bool follows = live && lane > 0 && slot == prev + 1 && (slot % kBlk8) != 0;
    const unsigned follow_mask = __ballot_sync(0xffffffffu, follows);
    const unsigned leaders = __ballot_sync(0xffffffffu, live && !follows && lane >= 1 && lane <= kAppendWindow);
    const int units = __popc(leaders) * a.c.H * 2;
    int odd = 0;
    for (int u = blockIdx.y * (kAppendWarps / W) + team; u < units; u += gridDim.y * (kAppendWarps / W), odd ^= 1) {
        const int hw = u % (a.c.H * 2), head = hw >> 1, which = hw & 1;
        unsigned rest = leaders;
        for (int k = u / (a.c.H * 2); k > 0; --k) rest &= rest - 1;
        const int lead = __ffs(rest) - 1;
        const unsigned behind = ~(follow_mask >> lead >> 1);       // bit j: entry lead + 1 + j does not follow
        const int m = 1 + (behind ? __ffs(behind) - 1 : 31);       // <= 16: the 17th would start a block
        const long long s0 = __shfl_sync(0xffffffffu, slot, lead);
        const long long page = s0 / kPage;
        const int in_page = (int)(s0 % kPage), off = in_page % kBlk8, blk = in_page / kBlk8;
        const T* src = static_cast<const T*>(which ? a.v : a.k);
        const long long stride = which ? a.v_stride : a.k_stride;
        int8_t* dst = a.c.pages + (((page * a.c.H + head) * 2 + which) * kPage + blk * kBlk8) * (long long)HD;
        float* sc = a.c.scales + ((page * a.c.H + head) * 2 + which) * kBlksPerPage + blk;
        const float s_old = off ? *sc : 0.f;
        float x[VPL][8];
        unsigned top = 0;                                           // bits of the largest magnitude: NaN above infinity above all else
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int e = i * TEAM + member, row = e / VPR;
            if (row < m) {
                load8(src + (long long)(t0 - 1 + lead + row) * stride + head * HD + (e % VPR) * 8, a.wide, x[i]);
#pragma unroll
                for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[i][j]) & 0x7fffffffu);
            }
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (W > 1) {                                                // the unit's other warp; the next unit writes the other half of s_top
            if (lane == 0) s_top[odd][warp] = top;
            asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(TEAM) : "memory");
            top = max(top, s_top[odd][warp ^ 1]);
        }
        float s = __fdiv_rn(__uint_as_float(top), 127.f);
        if (top) s = fmaxf(s, 1.17549435e-38f);
        const bool nan = top >= 0x7f800000u || s_old != s_old;
        s = nan ? __uint_as_float(0x7fffffffu) : fmaxf(s, s_old);
        const float inv = s > 0.f ? __frcp_rn(s) : 0.f;             // also 0 for NaN: compares false
        if (off && !(s == s_old)) {
            const double so = s_old, sn = s;
            for (int e = member; e < off * VPR; e += TEAM) {
                uint2 w = *reinterpret_cast<const uint2*>(dst + e * 8);
                int8_t* q = reinterpret_cast<int8_t*>(&w);
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = nan ? (int8_t)0 : (int8_t)__double2int_rn((double)q[j] * so / sn);
                *reinterpret_cast<uint2*>(dst + e * 8) = w;
            }
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int e = i * TEAM + member, row = e / VPR;
            if (row < m) *reinterpret_cast<uint2*>(dst + (off + row) * HD + (e % VPR) * 8) = nan ? make_uint2(0u, 0u) : quant8(x[i], s, inv);
        }
        if (member == 0) *sc = s;
    }
}

// ---- read back ------------------------------------------------------------------------------------------------------
struct Read8Args {
    Kv8View c;
    void* k; void* v;
    const long long* slots;
    long long k_stride, v_stride;
    int n_tok, wide;
};

// A block takes one head's K or V of kReadRows list entries, a thread eight values of four of them: rows of K and of V per
// entry, zeros for a slot outside the pool.  Bound by bytes (1 in, 2 or 4 out per value): 18 us for eight thousand rows of eight
// heads of 128 in fp32 (82 MB, 4.5 TB/s).
constexpr int kReadThreads = 256;
template <typename T, int HD>
__global__ void __launch_bounds__(kReadThreads) k_kv8_read(const Read8Args a) {
    constexpr int VPR = HD / 8, RPP = kReadThreads / VPR;        // threads per row, rows per pass
    pdl_wait();
    const int head = blockIdx.y >> 1, which = blockIdx.y & 1, vec = threadIdx.x % VPR;
    T* out = static_cast<T*>(which ? a.v : a.k) + head * HD + vec * 8;
    const long long stride = which ? a.v_stride : a.k_stride;
    const int t0 = blockIdx.x * RPP * 4 + threadIdx.x / VPR;
    long long run[4];
    int at[4];
    uint2 w[4];
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = t0 + i * RPP;
        const long long slot = t < a.n_tok ? a.slots[t] : -1;
        const bool in = slot >= 0 && slot < a.c.n_pages * kPage;
        run[i] = in ? ((slot / kPage) * a.c.H + head) * 2 + which : -1;
        at[i] = (int)(slot & (kPage - 1));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = make_uint2(0u, 0u); s[i] = 0.f;
        if (run[i] >= 0) {
            w[i] = *reinterpret_cast<const uint2*>(a.c.pages + (run[i] * kPage + at[i]) * HD + vec * 8);
            s[i] = a.c.scales[run[i] * kBlksPerPage + at[i] / kBlk8];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = t0 + i * RPP;
        if (t >= a.n_tok) continue;
        float f[8];
        const uint32_t u[2] = {w[i].x ^ 0x80808080u, w[i].y ^ 0x80808080u};
#pragma unroll
        for (int j = 0; j < 8; ++j)                              // a byte under 2^23: no conversion instruction
            f[j] = (__uint_as_float(__byte_perm(u[j >> 2], 0x4b000000u, 0x7440 + (j & 3))) - 8388736.f) * s[i];
        store8(out + t * stride, a.wide, f);
    }
}

}  // namespace sllm
