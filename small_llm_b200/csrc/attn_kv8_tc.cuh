// Attention over the 8-bit paged cache (kv8.cuh) for prompts: bf16 rows, head_dim 64 or 128, on the 5th-generation tensor cores.
//
// One block takes one kv head and NT tiles of 128 query rows (tokens x heads of the group) that follow on one another: two at
// head_dim 128, so that a key is widened once for 256 rows; one at 64, which leaves two blocks to an SM.  Per step, a page of 64 keys:
//   widening warps   int8 K and V from global memory (a step ahead, in registers) -> fp16 in shared memory, 128-byte swizzle
//   scales' warp     the four blocks' factors
//   MMA warp         S_t = Q_t K^T, 128 x 64 x hd, two steps ahead of the softmax, into one of two buffers;
//                    O_t += P_t V, 128 x hd x 64; both in tensor memory
//   softmax t        thread = query row = TMEM lane: w = exp2(...) as fp16 over S_t's own columns, where the next product reads it
//
// The integers are multiplied as they are (exact in fp16), scales act outside the products and cost nothing per element: with
// c = scale log2(e) ks(block) and v = vs(block) / vr the weight is  w = p v = exp2(S c + (log2 v - m)),  one fma and one ex2, and
// the softmax denominator sums w / v block by block.  vr is a power of two near the first vs, m the largest S c + log2 v so far less 7: what
// the attended values contribute, and not the loudest value of the cache, is what fp16's range is spent on, all of it: the largest
// weight is 2^7 or more, fp16 rounds one to 2^-11 of itself down to 2^-21 of the largest and drops it below 2^-32, so that what a hundred
// thousand keys beside a strong one add up to is kept.  (The output is rounded to bf16, 2^-8.)  q, bf16 divided by a power of two, is
// exact in fp16 down to 2^-16 of the row's largest value.  m does not follow every new
// maximum but one that brings weights above 2^15: O in tensor memory is then rescaled, which is rare,
// and so the exponentials need not wait for the maximum of their own step.
//
// What bounds it: 16 exponentials a clock and SM (1024 clocks for two tiles' step) against 1290 clocks of products at head_dim 128
// (S at 64 columns is bound by its operands' way through shared memory: 387 clocks where the products alone are 256).  Measured
// 2500 clocks a step: the three kinds of warps share the schedulers' issue slots.  On the way: one lane in a divergent loop, 128 keys
// a step and one S buffer 546 us, for 2770 new tokens x 32 heads of 128 behind 2000 to 6000 keys; roles with their own registers 296;
// two S buffers and 64 keys 281; weights beside their maximum, one body of code (masks go by way of S in tensor memory) 254; query rows read
// by lanes side by side 240 us, 850 TFLOP/s.  Tried and dropped: two threads per row (349 against 296), polls with a suspend hint (no difference), one tile per
// block at head_dim 128 (a step of 3100 tokens 89 us against 77 then).
// 7.4 thousand prompt tokens of ten heads of 64 take 44 us, half of it the blocks' beginnings and ends (eight steps on average).
// Where there are few blocks for the GPU the keys are cut into chunks (grid z), whose states the general form's second kernel joins.
// Every wait is bounded; on expiry the block sets *status, gives its rows NaN, frees its tensor memory and returns.
#pragma once
#include "attn_kv8.cuh"
#include "tc_ptx.cuh"

namespace sllm {

constexpr int kT8Rows = 128;                     // query rows of a tile
constexpr int kT8Keys = kPage;                   // keys of a step: a page
constexpr int kT8Blks = kT8Keys / kBlk8;         // scale blocks of a step
constexpr int kT8Ring = 8;                       // steps whose scales are held
constexpr int kT8Stages = 4;                     // widened K (and V) tiles
constexpr float kT8Start = 7.f;                  // log2 of a row's largest weight when m is set
constexpr float kT8Slack = 15.f;                 // log2 units that scores may pass m by: a weight is at most 2^15
constexpr int kT8MaxSort = 64;                   // sequences up to which blocks order the tiles by their keys
constexpr int kT8MaxCu = 1024;                   // sequences up to which a tile is looked for in shared memory

// NT tiles of query rows per block.  Warps: 4 NT softmax; 4 widening K and 4 widening V (NT = 1: 4 for both); the last four are
// the MMA warp, the scales' warp and two that idle.  Registers are dealt out again at the start (setmaxnreg).  In units of 128 threads, NT = 2:
// launched with 5 x 96 = 480; softmax 2 x 144, widening 2 x 72, the last four warps 48: 480.  NT = 1: 3 x 80 = 240; 136, 64, 40: 240.
template <int NT> __host__ __device__ constexpr int attn8_tc_threads() { return NT == 2 ? 640 : 384; }
constexpr int kT8BarBytes = 512;                 // barriers, and where the tensor memory begins
template <int HD, int NT> __host__ __device__ constexpr size_t attn8_tc_smem() {
    return 1024 + NT * (size_t)kT8Rows * HD * 2 + 2 * kT8Stages * (size_t)kT8Keys * HD * 2 + kT8Ring * (kT8Blks + 1) * 16 + kT8BarBytes;
}

__device__ __forceinline__ bool wait8(uint32_t bar, uint32_t parity) { return mbar_wait_bounded(bar, parity, kWaitLimitNs); }
// one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}
// Operand descriptors differ in their low words only, so those are what is kept and added to.
constexpr uint32_t kT8DescHi = (uint32_t)(64u | 1u << 14 | 2u << 29);
__device__ __forceinline__ uint32_t desc_lo(const void* p) { return ((smem_u32(p) >> 4) & 0x3fff) | 1u << 16; }
__device__ __forceinline__ void tc_mma_f16_ss(uint32_t tmem_d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 x, y;\nsetp.ne.b32 p, %4, 0;\nmov.b64 x, {%1, %5};\nmov.b64 y, {%2, %5};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}"
                 ::"r"(tmem_d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kT8DescHi) : "memory");
}
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 y;\nsetp.ne.b32 p, %4, 0;\nmov.b64 y, {%2, %5};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}"
                 ::"r"(tmem_d), "r"(tmem_a), "r"(b), "r"(idesc), "r"(acc), "n"(kT8DescHi) : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tc_ld32_async(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr));
}
// waits for the loads so far; the registers they fill pass through, so that no use of them moves in front of it
__device__ __forceinline__ void tc_wait_ld64(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 64; ++i) asm volatile("" : "+r"(r[i]));
}
// two floats at a time: a * b + c, a + b
__device__ __forceinline__ unsigned long long pair2(float a, float b) {
    unsigned long long x;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a), "f"(b));
    return x;
}
__device__ __forceinline__ float2 unpair2(unsigned long long x) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(x));
    return f;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int R> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }

template <int HD, int NT>
__global__ void __launch_bounds__(attn8_tc_threads<NT>(), NT == 1 ? 2 : 1) k_attn_kv8_tc(const Attn8Args a) {
    constexpr int SOFT = 4 * NT, WIDE = 4 * NT;               // softmax warps 0 .. SOFT - 1, then the widening ones, MMA, scales
    constexpr int THREADS = attn8_tc_threads<NT>();
    constexpr uint32_t TMEM_COLS = NT * (2 * kT8Keys + HD) > 256 ? 512 : 256;      // two S per tile, and O
    constexpr int HALVES = HD / 64;                           // 128-byte column blocks of a row
    constexpr uint32_t Q_HALF = kT8Rows * 128, HALF = kT8Keys * 128;       // bytes of one of them, of queries and of keys
    constexpr uint32_t Q_TILE = HALVES * Q_HALF, TILE = HALVES * HALF;
    constexpr int CPR = HD / 16;                              // 16-byte chunks of int8 per cache row
    constexpr int RPP = 128 / CPR;              // rows per pass of the widening threads
    constexpr int PASSES = kT8Keys / RPP;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* sQ = smem;                                       // [NT][Q_TILE]
    uint8_t* sK = sQ + NT * Q_TILE;                           // [stages][TILE]
    uint8_t* sV = sK + kT8Stages * TILE;
    float4* s_blk = reinterpret_cast<float4*>(sV + kT8Stages * TILE);      // [ring][blocks]: c, log2 v (-inf: does not count), 1 / v
    float4* s_vr = s_blk + kT8Ring * kT8Blks;                 // [ring]: vr
    uint64_t* bars = reinterpret_cast<uint64_t*>(s_vr + kT8Ring);
    // S_READY, P_READY and PV_DONE: [tile][step parity], for they may be a step ahead of who waits
    enum { K_FULL = 0, V_FULL = K_FULL + kT8Stages, K_FREE = V_FULL + kT8Stages, V_FREE = K_FREE + kT8Stages, S_READY = V_FREE + kT8Stages, P_READY = S_READY + 4,
           PV_DONE = P_READY + 4, SC_FULL = PV_DONE + 4, Q_FULL = SC_FULL + kT8Ring, N_BARS = Q_FULL + 1 };
    static_assert(N_BARS * 8 + 4 <= kT8BarBytes, "the barriers fit their place");
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + N_BARS);
    __shared__ int s_last[2][8];
    __shared__ int2 s_key[kT8MaxSort];                        // last position and tiles of each sequence
    __shared__ int s_cu[kT8MaxCu + 1];
    __shared__ int s_pick[2];
    __shared__ float s_rowf[NT][kT8Rows];
    const uint32_t bar0 = smem_u32(bars);
    auto B = [&](int i) { return bar0 + 8u * (uint32_t)i; };

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_launch_dependents();
    pdl_wait();
    // Which tile: those with the most keys first, so that the last blocks to start are short ones.  With few sequences each
    // block sorts them by their last position (the tiles of one are near one another); with many, the grid is long anyway.
    int t0 = 0, seq = 0, n = 0;
    if (a.n_seq <= kT8MaxSort) {
        if (tid == 0) s_pick[0] = -1;
        for (int i = tid; i < a.n_seq; i += THREADS) {
            const int c0 = a.cu_tok[i], c1 = min(a.cu_tok[i + 1], a.n_tok);
            const bool any = c0 >= 0 && c1 > c0;
            s_key[i] = make_int2(any ? a.tok_pos[c1 - 1] : -1, any ? (c1 - c0 + a.rows_toks - 1) / a.rows_toks : 0);
        }
        __syncthreads();
        for (int i = tid; i < a.n_seq; i += THREADS) {
            const int2 mine = s_key[i];
            int before = 0;
#pragma unroll 8
            for (int j = 0; j < a.n_seq; ++j) {
                const int2 k = s_key[j];
                before += (k.x > mine.x) | ((k.x == mine.x) & (j < i)) ? k.y : 0;
            }
            const int k = (int)blockIdx.y - before;
            if (k >= 0 && k < mine.y) { s_pick[0] = i; s_pick[1] = mine.y - 1 - k; }
        }
        __syncthreads();
        seq = s_pick[0];
        if (seq >= 0) {
            const int c0 = a.cu_tok[seq];
            t0 = c0 + s_pick[1] * a.rows_toks;
            n = min(a.rows_toks, min(a.cu_tok[seq + 1], a.n_tok) - t0);
        }
    } else {
        const bool fits = a.n_seq <= kT8MaxCu;
        if (fits) {
            for (int i = tid; i <= a.n_seq; i += THREADS) s_cu[i] = a.cu_tok[i];
            __syncthreads();
        }
        n = attn8_tile(a, fits ? s_cu : a.cu_tok, gridDim.y - 1 - blockIdx.y, t0, seq);
    }
    if (n <= 0) return;
    const int head = blockIdx.x, group = a.group, toks = a.rows_toks / NT;   // tokens of one tile
    const int most = (int)min((long long)a.width * kPage, 0x7fffff00ll) - 1;

    if (tid == 0) {
        for (int i = 0; i < kT8Stages; ++i) { mbar_init(B(K_FULL + i), 5); mbar_init(B(V_FULL + i), 4); mbar_init(B(K_FREE + i), 1); mbar_init(B(V_FREE + i), 1); }
        for (int i = 0; i < 4; ++i) { mbar_init(B(S_READY + i), 1); mbar_init(B(P_READY + i), 4); mbar_init(B(PV_DONE + i), 1); }
        for (int i = 0; i < kT8Ring; ++i) mbar_init(B(SC_FULL + i), 1);
        mbar_init(B(Q_FULL), SOFT);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == SOFT + WIDE) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // last position of each tile's tokens
    if (tid < 2 * kT8Rows) {
        int who = -1, at = -1;
        if (tid < n) { who = a.tok_seq[t0 + tid]; at = a.tok_pos[t0 + tid]; }
        const int pos = who == seq ? max(min(at, most), -1) : -1;            // an entry that does not name the sequence is skipped
        const int p0 = __reduce_max_sync(0xffffffffu, tid < toks ? pos : -1), p1 = __reduce_max_sync(0xffffffffu, tid < toks ? -1 : pos);
        if (lane == 0) { s_last[0][warp] = p0; s_last[1][warp] = p1; }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    int last0 = -1, last1 = -1;
#pragma unroll
    for (int i = 0; i < 8; ++i) { last0 = max(last0, s_last[0][i]); last1 = max(last1, s_last[1][i]); }
    // This block's chunk of the keys: from here on positions and pages count from its first key.  The last chunk takes all that is left.
    const int chunk = blockIdx.z, key0 = chunk * a.chunk, own_chunks = attn8_chunks(a, max(last0, last1));
    const int last = max(last0, last1) - key0, most_steps = chunk == a.n_chunks - 1 ? 0x7fffffff : a.chunk / kT8Keys;
    const int n0 = min(max(last0 - key0 + kT8Keys, 0) / kT8Keys, most_steps), n1 = min(max(last1 - key0 + kT8Keys, 0) / kT8Keys, most_steps);
    const int steps = max(n0, n1);                            // 0 where nothing is attended
    if (steps == 0 && chunk > 0) {                            // chunk 0 writes the rows that attend nothing
        if (warp == SOFT + WIDE) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS));
        return;
    }

    bool ok = true;

    const int* table = a.table + (size_t)seq * a.width + key0 / kPage;
    auto page_of = [&](int i) -> int {                        // page of a step; -2: outside the pool
        const int id = table[i];
        return id < 0 || id >= a.c.n_pages ? -2 : id;
    };
    auto parity = [](int i) { return (uint32_t)(i / kT8Stages) & 1u; };       // of step i's use of its stage
    if (warp >= SOFT + WIDE) {
        fewer_registers<NT == 2 ? 48 : 40>();
        if (warp == SOFT + WIDE) {
        // ---- MMA ----
        const uint32_t id_s = (1u << 4) | ((uint32_t)(kT8Keys >> 3) << 17) | ((uint32_t)(kT8Rows >> 4) << 24);     // fp16 x fp16 -> fp32
        const uint32_t id_o = (1u << 4) | (1u << 16) | ((uint32_t)(64 >> 3) << 17) | ((uint32_t)(kT8Rows >> 4) << 24);   // V: MN-major
        // descriptors of the first tiles; a place further on is its distance / 16 more
        const uint32_t q_desc = desc_lo(sQ), k_desc = desc_lo(sK), v_desc = desc_lo(sV);
        // One lane does it all: as few instructions as can be, for four busy warps share its scheduler.
        if (elect_one()) {
            auto issue_s = [&](int i, int t) {
                const uint32_t q = q_desc + (uint32_t)t * (Q_TILE / 16), k = k_desc + (uint32_t)(i % kT8Stages) * (TILE / 16);
                const uint32_t d = tmem + (uint32_t)((2 * t + (i & 1)) * kT8Keys);
#pragma unroll
                for (int j = 0; j < HD / 16; ++j)
                    tc_mma_f16_ss(d, q + ((j >> 2) * Q_HALF + (j & 3) * 32) / 16, k + ((j >> 2) * HALF + (j & 3) * 32) / 16, id_s, j != 0);
                tc_commit(B(S_READY + 2 * t + (i & 1)));
            };
            auto issue_o = [&](int i, int t) {
                const uint32_t v = v_desc + (uint32_t)(i % kT8Stages) * (TILE / 16), p = tmem + (uint32_t)((2 * t + (i & 1)) * kT8Keys);
#pragma unroll
                for (int h = 0; h < HALVES; ++h)
#pragma unroll
                    for (int j = 0; j < kT8Keys / 16; ++j)
                        tc_mma_f16_ts(tmem + NT * 2 * kT8Keys + t * HD + h * 64, p + j * 8, v + (h * HALF + j * 2048) / 16, id_o, i > 0 || j > 0);
                tc_commit(B(PV_DONE + 2 * t + (i & 1)));
            };
            // S runs two steps ahead of the softmax: it has the next step's scores when it ends one.  K_FULL stands for the scales
            // as well, which S does not need: so their warp, which K_FREE holds back, is never a whole phase of it behind.
            if (steps > 0) ok = wait8(B(Q_FULL), 0);
            for (int i = 0; i < 2 && i < steps && ok; ++i) {
                ok = wait8(B(K_FULL + i), 0);
                if (!ok) break;
                tc_fence_after();
                if (i < n0) issue_s(i, 0);
                if (i < n1) issue_s(i, 1);
                tc_commit(B(K_FREE + i));
            }
            for (int i = 0; i < steps && ok; ++i) {
                const int s = i % kT8Stages, s2 = (i + 2) % kT8Stages;
                ok = wait8(B(V_FULL + s), parity(i));
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int nt = t ? n1 : n0;
                    if (ok && i < nt) {
                        ok = wait8(B(P_READY + 2 * t + (i & 1)), (i >> 1) & 1);
                        tc_fence_after();
                        if (ok) issue_o(i, t);
                    }
                    if (t == 0 && ok && i + 2 < steps) {
                        ok = wait8(B(K_FULL + s2), parity(i + 2));
                        tc_fence_after();
                    }
                    if (ok && i + 2 < nt) issue_s(i + 2, t);
                }
                if (!ok) break;
                tc_commit(B(V_FREE + s));
                if (i + 2 < steps) tc_commit(B(K_FREE + s2));
            }
        }
        ok = __all_sync(0xffffffffu, ok);
        } else if (warp == SOFT + WIDE + 1) {
        // ---- the blocks' factors: lane b takes block b of a step; the loads are a step ahead ----
        float ks = 0.f, vs = 0.f, vr = 0.f;
        bool counts = false;
        int id = lane < kT8Blks && steps > 0 ? page_of(0) : -1;
        auto fetch = [&](int i) {
            counts = id >= 0 && (long long)i * kT8Keys + lane * kBlk8 <= last;
            if (id == -2 && a.status) atomicExch(a.status, 1);
            if (counts) {
                const float* sc = a.c.scales + ((long long)id * a.c.H + head) * 2 * kBlksPerPage + lane;
                ks = sc[0]; vs = sc[kBlksPerPage];
            }
        };
        if (steps > 0) fetch(0);
        for (int i = 0; i < steps && ok; ++i) {
            id = lane < kT8Blks && i + 1 < steps ? page_of(i + 1) : -1;
            float top = counts && vs < INFINITY ? vs : 0.f;          // one that is not finite is no reference
#pragma unroll
            for (int o = 1; o < kT8Blks; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (vr == 0.f && top > 0.f) vr = pow2_above(fminf(top, 1.7e38f));
            const float v0 = vr > 0.f ? vs / vr : (vs == 0.f ? 1.f : vs);
            // Within 2^-60 and 2^100: at the lower end fp16 takes a weight for 0 beside any other, the sum does not; the upper one is
            // out of reach for values that one model made.  A scale that is not finite makes the weights of its block NaN, and
            // nothing else: the other factors also meet rows that stand before it.
            const float v = fminf(fmaxf(v0, 8.67361738e-19f), 1.26765060e30f), odd = (ks - ks) + (vs - vs);       // 0 or NaN
            const float4 f = counts ? make_float4(ks * fabsf(a.scale) * 1.4426950408889634f, log2f(v) + odd, 1.f / v, 0.f) : make_float4(0.f, -INFINITY, 0.f, 0.f);
            // the K of a step is free once S is done, which was asked for when the softmax had ended the step two before: with the
            // K of step i - stages free it is done with i - stages - 2, far behind the ring's length
            if (i >= kT8Stages) ok = __all_sync(0xffffffffu, wait8(B(K_FREE + i % kT8Stages), parity(i - kT8Stages)));
            if (!ok) break;
            if (lane < kT8Blks) s_blk[(i % kT8Ring) * kT8Blks + lane] = f;
            if (lane == 0) s_vr[i % kT8Ring].x = vr;
            __syncwarp();
            if (lane == 0) { mbar_arrive(B(SC_FULL + i % kT8Ring)); mbar_arrive(B(K_FULL + i % kT8Stages)); }
            if (i + 1 < steps) fetch(i + 1);
        }
        }
    } else if (warp >= SOFT) {
        // ---- widening: int8 rows -> fp16 tiles, the loads a step ahead ----
        if constexpr (NT == 2) fewer_registers<72>(); else fewer_registers<64>();
        // A warp takes one 128-byte column block of eight rows: its lanes' stores, two rows of four chunks at a time, meet no bank twice.
        const int wi = warp & 3, c = (lane & 3) + (HALVES == 2 ? (wi >> 1) * 4 : 0), row0 = (lane >> 2) + (HALVES == 2 ? wi & 1 : wi) * 8;
        static_assert(RPP % 8 == 0, "rows of a thread share their place in the swizzle");
        const uint32_t at0 = (c >> 2) * HALF + sw128(row0, (2 * c) & 7), at1 = (c >> 2) * HALF + sw128(row0, ((2 * c) & 7) + 1);
        auto fetch = [&](int id, int which, uint4 (&x)[PASSES]) {
            const int8_t* src = a.c.pages + (((long long)id * a.c.H + head) * 2 + which) * (kPage * HD) + row0 * HD + c * 16;
#pragma unroll
            for (int j = 0; j < PASSES; ++j) x[j] = id >= 0 ? *reinterpret_cast<const uint4*>(src + j * RPP * HD) : make_uint4(0u, 0u, 0u, 0u);
        };
        auto widen = [&](uint8_t* dst, const uint4 (&x)[PASSES], int full) {
#pragma unroll
            for (int j = 0; j < PASSES; ++j) {
                const uint32_t u[4] = {x[j].x ^ 0x80808080u, x[j].y ^ 0x80808080u, x[j].z ^ 0x80808080u, x[j].w ^ 0x80808080u};
                const uint4 lo = make_uint4(halves(u[0], 0x4140), halves(u[0], 0x4342), halves(u[1], 0x4140), halves(u[1], 0x4342));
                const uint4 hi = make_uint4(halves(u[2], 0x4140), halves(u[2], 0x4342), halves(u[3], 0x4140), halves(u[3], 0x4342));
                *reinterpret_cast<uint4*>(dst + at0 + j * RPP * 128) = lo;
                *reinterpret_cast<uint4*>(dst + at1 + j * RPP * 128) = hi;
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(B(full));
        };
        auto freed = [&](int bar, int i) { return i < kT8Stages || __all_sync(0xffffffffu, wait8(B(bar + i % kT8Stages), parity(i - kT8Stages))); };
        if constexpr (NT == 2) {
            const int which = (warp - SOFT) >> 2;
            uint8_t* dst = which ? sV : sK;
            const int full = which ? V_FULL : K_FULL, free = which ? V_FREE : K_FREE;
            uint4 x[PASSES];
            int id = -1;
            if (steps > 0) fetch(page_of(0), which, x);
            if (steps > 1) id = page_of(1);
            for (int i = 0; i < steps && ok; ++i) {
                ok = freed(free, i);
                if (!ok) break;
                widen(dst + (i % kT8Stages) * TILE, x, full + i % kT8Stages);
                if (i + 1 < steps) fetch(id, which, x);
                if (i + 2 < steps) id = page_of(i + 2);
            }
        } else {
            uint4 xk[PASSES], xv[PASSES];
            int id = -1;
            if (steps > 0) { id = page_of(0); fetch(id, 0, xk); fetch(id, 1, xv); }
            if (steps > 1) id = page_of(1);
            for (int i = 0; i < steps && ok; ++i) {
                ok = freed(K_FREE, i);
                if (!ok) break;
                widen(sK + (i % kT8Stages) * TILE, xk, K_FULL + i % kT8Stages);
                if (i + 1 < steps) fetch(id, 0, xk);
                ok = freed(V_FREE, i);
                if (!ok) break;
                widen(sV + (i % kT8Stages) * TILE, xv, V_FULL + i % kT8Stages);
                if (i + 1 < steps) fetch(id, 1, xv);
                if (i + 2 < steps) id = page_of(i + 2);
            }
        }
    } else {
        // ---- softmax: thread = query row = TMEM lane ----
        if constexpr (NT == 2) more_registers<144>(); else more_registers<136>();
        // This thread's row; and the warp's 32 rows of q as fp16, K-major with the 128-byte swizzle, read and written by HD / 8 lanes each.
        // Rows of no token are zero.
        const int tile = warp >> 2, r = tid & 127;
        int pos = -1, row_tok = -1, row_head = 0;
        if (r / group < toks && tile * toks + r / group < n) {
            const int at = t0 + tile * toks + r / group, p = a.tok_pos[at];
            if (a.tok_seq[at] == seq) { row_tok = at; row_head = head * group + r % group; pos = max(min(p, most), -1) - key0; }     // tok_pos may be anything: no difference wraps
        }
        {
            constexpr int CH = HD / 8, RPI = 32 / CH;          // lanes per row, rows at a time
            const int c = lane % CH;
            const unsigned per = (65536u + group - 1) / group;  // rr / group = rr * per >> 16 for rr < 128
#pragma unroll 1
            for (int b = 0; b < CH; b += 8) {
                uint4 raw[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int rr = (r & ~31) + (b + i) * RPI + lane / CH, in = (int)((rr * per) >> 16), rt = tile * toks + in;
                    raw[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (in < toks && rt < n) {
                        const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(a.q) + (long long)(t0 + rt) * a.q_stride + (head * group + rr - in * group) * HD + c * 8;
                        if (a.wide) raw[i] = *reinterpret_cast<const uint4*>(src);
                        else {
                            uint32_t w[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) w[j] = (uint32_t)__bfloat16_as_ushort(src[2 * j]) | (uint32_t)__bfloat16_as_ushort(src[2 * j + 1]) << 16;
                            raw[i] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                }
                // rows whose maxima go through the shuffles side by side (all eight at head_dim 128: the registers that this takes from the steps
                // cost 5 %)
                constexpr int SIDE = HD == 64 ? 8 : 1;
#pragma unroll
                for (int i0 = 0; i0 < 8; i0 += SIDE) {
                    unsigned top[SIDE];
#pragma unroll
                    for (int i = 0; i < SIDE; ++i) {
                        const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw[i0 + i]);
                        top[i] = 0;
#pragma unroll
                        for (int j = 0; j < 4; ++j) top[i] = max(top[i], max((w[j] & 0x7fffu) << 16, w[j] & 0x7fff0000u));
                    }
#pragma unroll
                    for (int o = 1; o < CH; o <<= 1)
#pragma unroll
                        for (int i = 0; i < SIDE; ++i) top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
#pragma unroll
                    for (int i = 0; i < SIDE; ++i) {
                        const int rr = (r & ~31) + (b + i0 + i) * RPI + lane / CH;
                        // f = 2^-e with the largest value in [2^(e-1), 2^e), as in the general form
                        const int e = min(max((int)(top[i] >> 23) - 126, -125), 125);
                        const float f = top[i] ? __uint_as_float((uint32_t)(127 - e) << 23) : 1.f;
                        if (c == 0) s_rowf[tile][rr] = top[i] ? __uint_as_float((uint32_t)(127 + e) << 23) : 1.f;
                        const float fs = a.scale < 0.f ? -f : f;   // block factors are positive: a maximum may be taken before them
                        float x[8];
                        unpack16<__nv_bfloat16>(raw[i0 + i], x);
                        *reinterpret_cast<uint4*>(sQ + tile * Q_TILE + (c >> 3) * Q_HALF + sw128(rr, c & 7)) =
                            make_uint4(pack_half(x[0] * fs, x[1] * fs), pack_half(x[2] * fs, x[3] * fs), pack_half(x[4] * fs, x[5] * fs), pack_half(x[6] * fs, x[7] * fs));
                    }
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(B(Q_FULL));
        }
        const float row_f = s_rowf[tile][r];
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t o_at = lanes + NT * 2 * kT8Keys + tile * HD;
        const int my_steps = tile ? n1 : n0;
        const int open = row_tok >= 0 ? pos : 0x7fffffff;      // rows of no token, or of one that is skipped: whatever they come to is not written
        const int all_see = __reduce_min_sync(0xffffffffu, open);
        float m = -INFINITY, l = 0.f, vr = 0.f;
        // One step: the 64 scores of a row stay in registers.
        auto step = [&](int i) {
            const float4* blk = s_blk + (i % kT8Ring) * kT8Blks;
            const float vr_now = s_vr[i % kT8Ring].x;
            const uint32_t s_at = lanes + (uint32_t)((2 * tile + (i & 1)) * kT8Keys);
            const int k0 = i * kT8Keys;
            // In its first step a row needs a maximum to begin with; in its last one or two the keys behind it, which the block that its
            // own key lies in holds, get -inf in S.  (Whole blocks behind it do not count, see below.)
            const bool masked = k0 + kT8Keys - 1 > all_see;    // the same for the whole warp
            if (i == 0 || masked) {
                float mx = -INFINITY;
#pragma unroll 1
                for (int b = 0; b < kT8Blks; ++b) {
                    uint32_t x[16];
                    tc_ld16(s_at + b * 16, x);
                    float top = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        if (k0 + b * 16 + j > open) x[j] = 0xff800000u;
                        top = fmaxf(top, __uint_as_float(x[j]));
                    }
                    if (masked) tc_st16(s_at + b * 16, x);
                    mx = fmaxf(mx, fmaf(top, fmaxf(blk[b].x * row_f, 1e-37f), blk[b].y));
                }
                tc_wait_st();
                if (i == 0) { m = mx - kT8Start; vr = vr_now; }
            }
            // Weights against the m there is, and beside them their maximum, which the exponentials so need not wait for.  Where a row has
            // passed m by too much (in its first step, and rarely later), m moves and the step is done again: S is still there.
            uint32_t pk[32];
            float l_add;
            for (;;) {
                uint32_t sv[64];
                tc_ld32_async(s_at, sv);
                tc_ld32_async(s_at + 32, sv + 32);
                tc_wait_ld64(sv);
                const float m_use = m == -INFINITY ? 0.f : m;
                float mx = -INFINITY;
                l_add = 0.f;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    // c stays above zero, also beside a NaN, so that -inf stays -inf; a block behind the row does not count, whatever it holds: S
                    // is -inf there, and f.y, by which a scale that is not finite comes, is not used
                    const float4 f = blk[b];
                    const bool behind = k0 + b * 16 > open;
                    const float c = fmaxf(f.x * row_f, 1e-37f), d = behind ? -INFINITY : f.y - m_use;
                    float t4[2] = {__uint_as_float(sv[b * 16]), __uint_as_float(sv[b * 16 + 1])};
#pragma unroll
                    for (int j = 2; j < 16; j += 4) {
                        t4[0] = fmaxf(fmaxf(t4[0], __uint_as_float(sv[b * 16 + j])), __uint_as_float(sv[b * 16 + j + 1]));
                        if (j + 2 < 16) t4[1] = fmaxf(fmaxf(t4[1], __uint_as_float(sv[b * 16 + j + 2])), __uint_as_float(sv[b * 16 + j + 3]));
                    }
                    mx = fmaxf(mx, fmaf(fmaxf(t4[0], t4[1]), c, behind ? -INFINITY : f.y));
                    const unsigned long long c2 = pair2(c, c), d2 = pair2(d, d);
                    unsigned long long sum = 0;
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const float2 x = unpair2(fma2(pair2(__uint_as_float(sv[b * 16 + j]), __uint_as_float(sv[b * 16 + j + 1])), c2, d2));
                        const float w0 = exp2_fast(x.x), w1 = exp2_fast(x.y);
                        sum = add2(sum, pair2(w0, w1));
                        pk[b * 8 + j / 2] = pack_half(w0, w1);
                    }
                    const float2 s2 = unpair2(sum);
                    l_add = fmaf(s2.x + s2.y, f.z, l_add);
                }
                const bool moves = mx > m + kT8Slack || (m == -INFINITY && mx > m);
                if (!__any_sync(0xffffffffu, moves || vr_now != vr)) break;
                const float m_new = moves ? mx - kT8Start : m;
                const float corr = m == -INFINITY ? 0.f : exp2_fast(m - m_new);
                l *= corr;
                if (i > 0) {                                   // O as the products so far leave it: the last of them has to be done
                    if (ok) ok = wait8(B(PV_DONE + 2 * tile + ((i - 1) & 1)), ((i - 1) >> 1) & 1);
                    ok = __all_sync(0xffffffffu, ok);
                    tc_fence_after();
                    const float f = corr * (vr_now > 0.f ? vr / vr_now : 1.f);
#pragma unroll 1
                    for (int c = 0; c < HD / 16; ++c) {
                        uint32_t x[16];
                        tc_ld16(o_at + c * 16, x);
#pragma unroll
                        for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * f);
                        tc_st16(o_at + c * 16, x);
                    }
                }
                m = m_new;
                vr = vr_now;
            }
            l += l_add;
            tc_st16(s_at, pk);                                 // over columns of S that this thread has read
            tc_st16(s_at + 16, pk + 16);
        };
        for (int i = 0; i < my_steps && ok; ++i) {
            ok = wait8(B(SC_FULL + i % kT8Ring), (i / kT8Ring) & 1) && wait8(B(S_READY + 2 * tile + (i & 1)), (i >> 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            step(i);
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(B(P_READY + 2 * tile + (i & 1)));
        }
        if (my_steps > 0 && ok) ok = wait8(B(PV_DONE + 2 * tile + ((my_steps - 1) & 1)), ((my_steps - 1) >> 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        if (!ok) l = __uint_as_float(0x7fffffffu);             // a wait ran out: the rows become NaN
        const bool whole = own_chunks <= 1;
        const float f = whole ? (l == 0.f ? 0.f : vr / l) : l == l ? vr : l;
        const long long part = ((long long)row_tok * a.n_heads + row_head) * a.n_chunks + chunk;
        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + (row_tok >= 0 ? (long long)row_tok * a.out_stride + row_head * HD : 0);
        if (!whole && row_tok >= 0) { a.part_ml[part * 2] = m; a.part_ml[part * 2 + 1] = l; }
#pragma unroll
        for (int h = 0; h < HD / 16; ++h) {
            uint32_t o[16];
            if (my_steps > 0) tc_ld16(o_at + h * 16, o);
            float x[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = l == 0.f || my_steps == 0 ? 0.f : __uint_as_float(o[j]) * f;
            if (row_tok < 0) continue;
            if (whole) { store8(dst + h * 16, a.wide, x); store8(dst + h * 16 + 8, a.wide, x + 8); }
            else { store8(a.part + part * HD + h * 16, true, x); store8(a.part + part * HD + h * 16 + 8, true, x + 8); }
        }
    }
    if (!ok && a.status) atomicExch(a.status, 5);
    tc_fence_before();
    __syncthreads();
    if (warp == SOFT + WIDE) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS));
    }
}

}  // namespace sllm
