// Prompt attention over a cache of keys and values in 4 bits (packed_kv.cuh) on the tcgen05 tensor cores: ragged, causal, with or without a
// window, bfloat16, head sizes 64 and 128.
//
// A CTA takes GROUPS · 128 consecutive new tokens of one sequence and one head and walks the keys they see in blocks of 64 up to the
// diagonal.  Its warps have fixed jobs:
//   producers      codes and pairs of a block from the cache into registers, a block ahead; from there zero + step · code as float16 into a ring of 64 KB of
//                  shared memory, K and V in turn, in the 128-byte swizzle that the MMA reads.  A code becomes a number by a mask under an exponent, two
//                  at a time; pairs of entries i and i + 4 of eight stay neighbours, so the numbers of a row lie permuted, those of the queries likewise (the
//                  sum does not care), and the result is put in order where it is written.  Rows that no query may see, behind the sequence's last
//                  token or in blocks wholly before the window, are zeros and are not read;
//   MMA warps      (one a group) S = Q·Kᵀ into tensor memory and, once the probabilities are there, O += P·V (P is the operand in tensor memory, V
//                  is read as it lies, head dimension contiguous);
//   softmax warps  eight a group of 128 queries: a query is one lane of tensor memory, and two threads have a half of a block's keys each;
//                  running maximum and sum in float32, O scaled where a maximum grew.
// With GROUPS = 2 two groups share every block that the producers take apart.
//
// Queries, keys, weights and values are float16 operands (11 bits: each off by up to 2^-11 of itself), scores, sums and results float32; as bfloat16 they
// together moved a result by 2.5 times what its own rounding does, as float16 by a tenth of that.  What float16 lacks in range powers of two give: the
// queries' from their largest, the keys' and the values' from the CTA's first block, weights stay below 2^15; a key or a value 2^14 times as large as
// the first block's, or 2^-10, gets a power of its own, which costs its block a slower pass: what a query attends is as exact whatever the first block
// holds, which, with a window, it may not see.
// A value that is not a number must not meet the weight 0 of a query that does not see it (0 · NaN is not 0): its row of V becomes zeros, and its
// key's row of K NaN instead, which the mask hides from the same queries; so a head's row that sees it is NaN throughout.
//
// Bound by the chain of a block, some 2,800 cycles at head size 128 of which the tensor cores have 1,000: producers take a block's numbers apart in the issue
// slots that softmax leaves (1,000 cycles each for K and V), and S waits for them.  More producers would take registers from the softmax warps (28 warps: 173 us
// where 22 took 119); blocks of 64 keys with two threads a row are what 80 registers hold, all but 28 to 138 bytes of a thread that are spilled.  Measured: 512 new
// tokens behind 7500, 32 heads of 128 over 8: 123 us, 0.53 PFLOP/s (of them 2 for looking for small keys and values, 2.5 for the tile's place in scratch); twice
// 1024 new tokens, 12 heads of 64: 22.1 us.
// Every wait is bounded; a CTA that gives up sets the device error word, waits (bounded) for its MMAs, frees its tensor memory and leaves.
#include <type_traits>
#include <cuda_fp16.h>
#include "common.cuh"
#include "packed_kv.cuh"
#include "tcgen05.cuh"

namespace {
constexpr int PP_CB = 64, PP_BK = 64, PP_RING = 65536;              // tokens of a cache block; keys of a block; bytes of the ring
constexpr int PP_MAX_PARTS = 16;
constexpr int PP_FAR = 80;                                          // powers of their own of small keys and values: 2^-80 of the first block's at least
// Weights lie 2^PP_UP times as large (float16 then has them down to 2^-28 of the reference point's), and add up to PP_MOST at most before that moves: any is
// float16 still.  (32 weights that add up to 2^15: one is 2^10 at least, 2^6 above the reference point's.)
constexpr float PP_UP = 4.f, PP_MOST = 32768.f, PP_LEAST = 5.f;
constexpr __host__ __device__ int pp_producers(int GROUPS) { return 2 * GROUPS; }
constexpr __host__ __device__ int pp_threads(int GROUPS) { return (GROUPS * 8 + pp_producers(GROUPS) + GROUPS) * 32; }
constexpr __host__ __device__ int pp_part_floats(int DH) { return DH * 128 + 256; }

__device__ __forceinline__ float pp_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two float32 numbers that go through one instruction (sm_100)
__device__ __forceinline__ uint64_t pp_two(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ void pp_apart(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t pp_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t pp_add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// MN-major tile: rows of 64 elements (128 bytes, swizzled) are the operand's N, a row a step of its K; groups of 8 rows 1024 bytes apart, chunks of
// 64 along N `chunk` bytes apart
__device__ __forceinline__ uint64_t pp_desc_mn(const void* tile, uint32_t chunk) {
    uint64_t d = 0;
    d |= (uint64_t)((tsm(tile) >> 4) & 0x3FFF);
    d |= (uint64_t)(chunk >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// instruction descriptor: D float32, A and B float16, A K-major, B K-major or (mn) MN-major
__host__ __device__ constexpr uint32_t pp_idesc(int M, int N, bool mn) {
    return (1u << 4) | (mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void pp_mma_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void pp_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void pp_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
// Eight codes of a word as float16 numbers step · code + zero, entries (0, 4), (1, 5), (2, 6), (3, 7): a code under the exponent of 1024, where the upper
// code of a byte counts sixteenfold, so half of the shifts go.
__device__ __forceinline__ uint4 pp_numbers(uint32_t w, __half2 step, __half2 zero) {
    const __half2 less = __float2half2_rn(-1024.f), by = __float2half2_rn(0.0625f), less16 = __float2half2_rn(-64.f);
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t x = w >> (8 * i), lo = (x & PK_LOW) | 0x64006400u, hi = (x & PK_HIGH) | 0x64006400u;
        const __half2 a = __hfma2(__hadd2(*reinterpret_cast<const __half2*>(&lo), less), step, zero);
        const __half2 b = __hfma2(__hfma2(*reinterpret_cast<const __half2*>(&hi), by, less16), step, zero);
        r[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
        r[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}
// 2^e, e held to what float32 has
__device__ __forceinline__ float pp_power(int e) { return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23); }
// the exponent of a bfloat16 (of the bits of its upper half, sign away): 2^e ≤ |x| < 2^(e + 1); −127 for zero and what is below 2^-126
__device__ __forceinline__ int pp_exponent(uint32_t bits) { return (int)(bits >> 7 & 255u) - 127; }

// what the queries are divided by, as a power of two: their largest (its bits) comes to 2^14
__device__ __forceinline__ int pp_up(uint32_t top) { return max(pp_exponent(top), -110) - 14; }

template <int DH, int GROUPS>
__global__ void __launch_bounds__(pp_threads(GROUPS), GROUPS == 1 ? 2 : 1)
attn_packed_prefill_kernel(const __nv_bfloat16* __restrict__ qkv, int ld, int q_off, const unsigned char* __restrict__ Kq, const uint32_t* __restrict__ Kp,
                           const unsigned char* __restrict__ Vq, const uint32_t* __restrict__ Vp, int n_blocks, const int* __restrict__ block_table,
                           int max_blocks, const int* __restrict__ seq_slot, const int* __restrict__ seq_start, const int* __restrict__ seq_pos0,
                           __nv_bfloat16* __restrict__ out, int ld_out, int H, int Hkv, float scale, int window, int n_parts, int part_blocks, float* __restrict__ partials,
                           int* __restrict__ counters, int n_tiles, int n_seqs, int n_flat, int n_places, int least_new, int* __restrict__ dev_err) {
    constexpr int BK = PP_BK, PP_TILE = BK * DH * 2, PP_SLOTS = PP_RING / PP_TILE, ROWS = GROUPS * 128, NG = DH / 64, NPROD = pp_producers(GROUPS), SOFT = GROUPS * 8;
    constexpr int Q_BYTES = 128 * DH * 2, ATOM_Q = 16384, ATOM_KV = BK * 128;    // a 64-number chunk of 128 queries / of a block
    constexpr int NP = BK + DH + BK <= 256 ? 2 : 1;                 // buffers of P that a group's 256 columns have room for
    constexpr int HK = BK / 2, NC = HK / 32, HD = DH / 2;           // keys, chunks of 32 keys, and columns of O of a softmax thread
    extern __shared__ unsigned char pp_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(pp_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* q_tiles = smem;                                  // [GROUPS][NG][128][128 B]
    unsigned char* kv_tiles = smem + GROUPS * Q_BYTES;              // [PP_SLOTS][NG][BK][128 B]: K_0, V_0, K_1, V_1, …
    float* s_part = reinterpret_cast<float*>(kv_tiles + PP_RING);     // [GROUPS][2][128]
    float2* s_far = reinterpret_cast<float2*>(s_part + GROUPS * 256);            // [PP_SLOTS][64]: of block b at b % PP_SLOTS, each key's powers (see producers)
    uint32_t* s_any_far = reinterpret_cast<uint32_t*>(s_far + PP_SLOTS * 64);    // [PP_SLOTS]: whether any of a producer's is not 0, a byte each (without: not written)
    uint64_t* q_known = reinterpret_cast<uint64_t*>(s_any_far + PP_SLOTS);
    uint64_t* q_full = q_known + 1;       // [GROUPS]
    uint64_t* full = q_full + GROUPS;
    uint64_t* empty = full + PP_SLOTS;
    uint64_t* s_full = empty + PP_SLOTS;                            // [GROUPS] each from here
    uint64_t* s_read = s_full + GROUPS;
    uint64_t* p_full = s_read + GROUPS;                             // [GROUPS][NP], product i at i % NP: either side may be NP − 1 blocks ahead
    uint64_t* o_full = p_full + GROUPS * NP;
    uint64_t* drained = o_full + GROUPS * NP;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
    int* s_abort = reinterpret_cast<int*>(tmem_slot + 1);
    int* s_never = s_abort + 1;                                     // stays 0: for waits that nothing calls off
    int* s_top = s_never + 1;                                       // the largest of the queries' bits, sign away
    int* s_first = s_top + 1;                                       // [2]: of the largest numbers of the first block's keys and of its values, the smallest, as bits
    float* s_unit = reinterpret_cast<float*>(s_first + 2);          // [2]: from an MMA's result to a score in units of log2(e); from one of O to a number
    int* s_last = reinterpret_cast<int*>(s_unit + 2);                                        // [GROUPS]: whether this CTA merges its tile's parts
    int* s_place = s_last + GROUPS;                                 // the tile's place in scratch

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < PP_SLOTS; ++i) { tbar_init(&full[i], NPROD); tbar_init(&empty[i], GROUPS); }
        for (int g = 0; g < GROUPS; ++g) {
            tbar_init(&q_full[g], 8);
            tbar_init(&s_full[g], 2);                               // the MMAs, and what the producers left beside the numbers
            tbar_init(&s_read[g], 8);
            for (int i = 0; i < NP; ++i) { tbar_init(&p_full[g * NP + i], 8); tbar_init(&o_full[g * NP + i], 1); }
            s_last[g] = 1;
        }
        tbar_init(drained, GROUPS);
        tbar_init(q_known, SOFT);
        *s_abort = 0;
        *s_never = 0;
        *s_top = 0;
        s_first[0] = s_first[1] = 0x7f80;
        for (int i = 0; i < PP_SLOTS; ++i) s_any_far[i] = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    // z is the slowest index of the order in which CTAs are started: first parts first, and within a part long tiles first
    const int h = blockIdx.x;
    int part, qt, seq;
    if (n_flat == 0) {
        part = blockIdx.z / n_tiles;
        qt = n_tiles - 1 - blockIdx.z % n_tiles;
        seq = blockIdx.y;
    } else {
        // sequences of very unequal numbers of new tokens: the grid has as many places as their tiles can need, and place f is the f-th tile there is
        part = blockIdx.z / n_flat;
        int f = blockIdx.z % n_flat;
        seq = -1;
        qt = 0;
        for (int s0 = 0; s0 < n_seqs && seq < 0; s0 += 32) {        // (every warp looks; the answer is the same)
            const int s = s0 + lane, len = s < n_seqs ? seq_start[s + 1] - seq_start[s] : 0, tiles = len >= least_new ? min((len + ROWS - 1) / ROWS, n_tiles) : 0;
            int upto = tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int from = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += from;
            }
            const uint32_t behind = __ballot_sync(0xffffffffu, f < upto);
            if (behind != 0u) {
                const int l = __ffs(behind) - 1;
                seq = s0 + l;
                qt = __shfl_sync(0xffffffffu, upto, l) - 1 - f;     // (its long tiles first)
            } else {
                f -= __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        if (seq < 0) return;                                        // (more places than tiles; uniform over the CTA)
    }
    const int row0 = seq_start[seq], n_new = seq_start[seq + 1] - row0, slot = seq_slot[seq], pos0 = seq_pos0[seq];
    const int hk = h / (H / Hkv);
    const int t_first = qt * ROWS, q_first = pos0 + t_first;        // the tile's first query, in the step and in the sequence
    const int n_rows = min(n_new - t_first, ROWS), q_last = q_first + n_rows - 1;
    const int first_key = window > 0 ? max(0, q_first - window + 1) : 0;
    const int kb_first = first_key / BK, n_kb = q_last / BK - kb_first + 1;
    // the tile's key blocks are dealt to tile_parts CTAs, of part_blocks each or more; the others of its n_parts have nothing to do
    int tile_parts = max(1, min(n_parts, (n_kb + part_blocks - 1) / part_blocks));
    if (tile_parts > 1) {
        // Scratch has places for tiles that reach part_blocks blocks or more from their sequence's first token only, which are its last ones: this tile's is
        // behind those of the sequences before.  (Where there is none left the tile is not dealt; uniform over the CTA.)
        const int whole = min(part_blocks, 1 << 24) * BK;           // tokens that a CTA takes by itself whatever the rest
        int place = min((n_new + ROWS - 1) / ROWS, n_tiles) - 1 - qt;
        for (int s0 = 0; s0 < seq; s0 += 32) {
            const int s = s0 + lane, len = s < seq ? seq_start[s + 1] - seq_start[s] : 0, tiles = len >= least_new ? min((len + ROWS - 1) / ROWS, n_tiles) : 0;
            const int alone = tiles > 0 ? whole - seq_pos0[s] : len;             // new tokens that end before that many positions
            place += (int)__reduce_add_sync(0xffffffffu, (unsigned)(alone < len ? max(tiles - max(alone, 0) / ROWS, 0) : 0));
        }
        if (place >= n_places) tile_parts = 1;
        if (threadIdx.x == 0) *s_place = place;
    }
    const bool active = n_rows > 0 && n_new >= least_new && slot >= 0 && pos0 >= 0 && part < tile_parts;      // uniform over the CTA
    if (!active) return;                                            // (before it holds anything)
    constexpr uint32_t TMEM_COLS = 256 * GROUPS;                    // a group: S BK columns, O DH, P NP times BK / 2 (two float16 a column)
    if (warp == SOFT) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tsm(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const int my_first = kb_first + (int)((long long)part * n_kb / tile_parts);
    const int my_n = kb_first + (int)((long long)(part + 1) * n_kb / tile_parts) - my_first, my_end = my_first + my_n;
    // the blocks of group g: lo … hi − 1 (a group without rows: none)
    int lo[GROUPS], hi[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        const int qf = q_first + g * 128, rows = min(n_rows - g * 128, 128);
        lo[g] = max(my_first, (window > 0 ? max(0, qf - window + 1) : 0) / BK);
        hi[g] = rows > 0 ? min(my_end, (qf + rows - 1) / BK + 1) : lo[g];
        hi[g] = my_n > 0 ? max(hi[g], lo[g]) : lo[g];
    }
    const int* table = block_table + (size_t)max(slot, 0) * max_blocks;

    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;

    if (warp >= SOFT && warp < SOFT + NPROD) {
        // ---- producers: warp p has rows p · PR … of every block
        constexpr int PR = BK / NPROD, UNITS = PR * (DH / 32) / 32; // a unit: 32 entries of a row (16 bytes of codes); so many a lane
        const int p = warp - SOFT;
        const int n_exist = pos0 + n_new;                           // tokens that the cache holds
        struct Piece { uint4 codes[UNITS]; uint32_t pairs[UNITS], value_pairs[UNITS]; } piece[2];   // of the next K tile and the next V tile
        int held = -1;                                              // the cache blocks of 32 blocks at a time lie a lane each
        auto block_of = [&](int b) {
            if ((b & 31) == 0) {
                const int k0 = (my_first + b + lane) * BK + p * PR, cb = k0 / PP_CB;         // (a warp's rows lie in one cache block)
                const bool wanted = b + lane < my_n && k0 < n_exist && (cb + 1) * PP_CB > first_key;
                held = wanted ? packed_block(table, max_blocks, n_blocks, cb) : -1;
                if (wanted && held < 0) atomicOr(dev_err, VLRF_DEVERR_NO_BLOCK);
            }
            return __shfl_sync(0xffffffffu, held, b & 31);
        };
        auto fetch = [&](int b, int blk, auto value_c, Piece& into) {
            constexpr bool VALUE = decltype(value_c)::value;
            const int k0 = (my_first + b) * BK + p * PR;
            const size_t at = ((size_t)max(blk, 0) * Hkv + hk) * PP_CB + k0 % PP_CB;
#pragma unroll
            for (int i = 0; i < UNITS; ++i) {
                const int u = i * 32 + lane, r = u / (DH / 32), c = u % (DH / 32);
                into.codes[i] = make_uint4(0u, 0u, 0u, 0u);
                into.pairs[i] = into.value_pairs[i] = 0u;
                if (blk >= 0 && k0 + r < n_exist) {
                    into.codes[i] = *reinterpret_cast<const uint4*>((VALUE ? Vq : Kq) + (at + r) * (DH / 2) + c * 16);
                    into.value_pairs[i] = Vp[(at + r) * NG + c / 2];
                    if (!VALUE) into.pairs[i] = Kp[(at + r) * NG + c / 2];
                }
            }
        };
        // Keys and values lie divided by powers of two, 2^key_up and 2^value_up, that take to 1 … 2 the smallest of the largest numbers that the keys, or the
        // values, of the CTA's first block have each.  Numbers up to 2^15 times that are float16 then, and those of a row whose largest is 2^-10 of it are off by
        // 2^-11 of that largest (15 steps by 2^-25 each).  A key or a value beyond, either way (`far`), lies divided by a power of its own; its score is
        // multiplied, or its weight, by what that is more or less: the reference point is one of weights times powers, so the weights keep their bits.  (No
        // less than 2^-PP_FAR, so that sums of weights alone are float32 numbers.)
        int key_up = 0, value_up = 0;
        auto top_of = [](uint32_t pair) {                           // the largest number of a group, as bits of a bfloat16 (NaN: 0)
            const float zero = pair_zero(pair), top = fmaxf(fabsf(zero), fabsf(fmaf(15.f, pair_step(pair), zero)));
            return top == top ? (int)(__float_as_uint(top) >> 16) : 0;
        };
        auto both = [](int e) { return NG == 2 ? max(e, __shfl_xor_sync(0xffffffffu, e, 2)) : e; };     // (a row's other group is two lanes on)
        int value_far[UNITS];                                       // of the block that is being put
        // a pair whose zero is below 2^14 and whose step is below 2^10 times the unit needs no power of its own (|zero| + 15 step < 2^15), nor does one whose
        // zero is 2^-10 of it or more; both as bfloat16, the zero's in the upper half, so that words compare as their zeros do
        uint32_t key_limit = 0u, value_limit = 0u;
        auto limit_of = [](int up) { return (uint32_t)(up + 10 + 127) << 7 | (uint32_t)(up + 14 + 127) << 23; };
        auto floor_of = [](uint32_t limit) { return limit - (24u << 23); };     // (2^14 to 2^-10)
        auto beyond = [](uint32_t most, uint32_t limit) {           // (NaN is not)
            const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&most), b = *reinterpret_cast<const __nv_bfloat162*>(&limit);
            return __hge(a.x, b.x) || __hge(a.y, b.y);
        };
        auto larger = [](uint32_t x, uint32_t y) {                  // of both halves, signs away
            x &= 0x7fff7fffu;
            const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
            return *reinterpret_cast<const uint32_t*>(&m);
        };
        auto far_of = [&](uint32_t pair, int up) {
            const int top = both(top_of(pair)), e = pp_exponent((uint32_t)top) - up;
            return e > 14 ? e - 14 : e < -10 && top != 0 ? max(e, -PP_FAR) : 0;
        };
        auto put = [&](int t, const Piece& from) -> bool {          // tile t of this CTA: block t / 2, K or V
            const int sl = t % PP_SLOTS, use = t / PP_SLOTS;
            int key_far[UNITS];
            bool any = false;
#pragma unroll
            for (int i = 0; i < UNITS; ++i) key_far[i] = 0;
            if (!(t & 1)) {
                uint32_t key_most = 0u, value_most = 0u, key_least = 0xffffffffu, value_least = 0xffffffffu;
#pragma unroll
                for (int i = 0; i < UNITS; ++i) {
                    value_far[i] = 0;
                    key_most = larger(from.pairs[i], key_most);
                    value_most = larger(from.value_pairs[i], value_most);
                    key_least = min(key_least, from.pairs[i] & 0x7fff7fffu);
                    value_least = min(value_least, from.value_pairs[i] & 0x7fff7fffu);
                }
                any = __any_sync(0xffffffffu, beyond(key_most, key_limit) || beyond(value_most, value_limit) || key_least < floor_of(key_limit) ||
                                                  value_least < floor_of(value_limit));
            }
            if (any) {
                int most = 0;
#pragma unroll
                for (int i = 0; i < UNITS; ++i) {
                    key_far[i] = far_of(from.pairs[i], key_up);
                    value_far[i] = far_of(from.value_pairs[i], value_up);
                    most |= key_far[i] | value_far[i];
                }
                any = __any_sync(0xffffffffu, most != 0);           // (a zero may be small in a row that is not, or where nothing is)
            }
            __half2 step[UNITS], zero[UNITS];
#pragma unroll
            for (int i = 0; i < UNITS; ++i) {
                const bool nan_value = (from.value_pairs[i] & 0x7fffu) > 0x7f80u;        // (NaN in a value's pair, both halves of it: zeros in V, NaN in K)
                const uint32_t pair = (t & 1) ? (nan_value ? 0u : from.value_pairs[i]) : (nan_value ? 0x7fff7fffu : from.pairs[i]);
                const float down = pp_power(-((t & 1) ? value_up + value_far[i] : key_up + key_far[i]));
                step[i] = __float2half2_rn(pair_step(pair) * down);
                zero[i] = __float2half2_rn(pair_zero(pair) * down);
            }
            if (use >= 1 && !tbar_wait_warp(&empty[sl], (uint32_t)((use - 1) & 1), s_abort)) return false;
            unsigned char* tile = kv_tiles + (size_t)sl * PP_TILE;
            if (!(t & 1)) {
                const int at = t / 2 % PP_SLOTS;
                if (any) {
#pragma unroll
                    for (int i = 0; i < UNITS; ++i) {
                        const int u = i * 32 + lane, r = p * PR + u / (DH / 32), c = u % (DH / 32);
                        if (c == 0) s_far[at * 64 + r] = make_float2(pp_power(key_far[i]), (float)value_far[i]);
                    }
                }
                if (lane == 0) reinterpret_cast<unsigned char*>(s_any_far + at)[p] = any;
            }
#pragma unroll
            for (int i = 0; i < UNITS; ++i) {
                const int u = i * 32 + lane, r = p * PR + u / (DH / 32), c = u % (DH / 32);
                unsigned char* dst = tile + (c >> 1) * ATOM_KV + r * 128;
                const uint32_t w[4] = {from.codes[i].x, from.codes[i].y, from.codes[i].z, from.codes[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(dst + ((((c & 1) * 4 + j) ^ (r & 7)) << 4)) = pp_numbers(w[j], step[i], zero[i]);
            }
            return true;
        };
        auto hand_over = [&](int t) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");         // the MMA reads them
            __syncwarp();
            if (lane == 0) tbar_arrive(&full[t % PP_SLOTS]);
        };
        bool ok = true;
        if (my_n > 0) {
            const int blk = block_of(0);
            fetch(0, blk, std::false_type{}, piece[0]);
            fetch(0, blk, std::true_type{}, piece[1]);
            uint32_t top[2] = {0x7f80u, 0x7f80u};
#pragma unroll
            for (int i = 0; i < UNITS; ++i) {
                const uint32_t a = (uint32_t)both(top_of(piece[0].pairs[i])), b = (uint32_t)both(top_of(piece[1].value_pairs[i]));
                top[0] = min(top[0], a != 0 ? a : 0x7f80u);         // (a row of zeros says nothing)
                top[1] = min(top[1], b != 0 ? b : 0x7f80u);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                top[x] = __reduce_min_sync(0xffffffffu, top[x]);
                if (lane == 0) atomicMin(&s_first[x], (int)top[x]);
            }
            asm volatile("bar.sync 11, %0;" ::"n"(NPROD * 32) : "memory");
            // (where no row says anything: 2^0; the top of float32 is kept away from, so that sums of weights times values have room)
            key_up = s_first[0] == 0x7f80 ? 0 : min(max(pp_exponent((uint32_t)s_first[0]), -110), 80);
            value_up = s_first[1] == 0x7f80 ? 0 : min(max(pp_exponent((uint32_t)s_first[1]), -110), 80);
            key_limit = limit_of(key_up);
            value_limit = limit_of(value_up);
            ok = tbar_wait_warp(q_known, 0, s_abort);
            if (p == 0 && lane == 0) {
                s_unit[0] = fminf(pp_power(key_up) * (scale * 1.4426950408889634f) * pp_power(pp_up((uint32_t)*s_top)), 3.4028235e38f);
                s_unit[1] = pp_power(value_up);
            }
        }
        for (int b = 0; b < my_n && ok; ++b) {
            const int next = b + 1 < my_n ? block_of(b + 1) : -1;
            if (!(ok = put(2 * b, piece[0]))) break;
            hand_over(2 * b);
            if (b + 1 < my_n) fetch(b + 1, next, std::false_type{}, piece[0]);
            if (!(ok = put(2 * b + 1, piece[1]))) break;
            hand_over(2 * b + 1);
            if (b + 1 < my_n) fetch(b + 1, next, std::true_type{}, piece[1]);
        }
        if (!ok) atomicExch(s_abort, 1);
    } else if (warp >= SOFT + NPROD) {
        // ---- MMAs, a warp a group
        const int g = warp - SOFT - NPROD, my_lo = g == 0 ? lo[0] : lo[GROUPS - 1], my_hi = g == 0 ? hi[0] : hi[GROUPS - 1];
        constexpr uint32_t idesc_s = pp_idesc(128, BK, false), idesc_o = pp_idesc(128, DH, true);
        const uint64_t dq = umma_desc_k128(q_tiles + g * Q_BYTES), dk0 = umma_desc_k128(kv_tiles), dv0 = pp_desc_mn(kv_tiles, ATOM_KV);
        const uint32_t tmem_s = tmem + g * 256, tmem_o = tmem_s + BK, tmem_p = tmem_o + DH;
        bool ok = true;
        // S_j = Q · K_jᵀ where the group sees block j; either way the group is done with K_j then
        auto issue_s = [&](int j) -> bool {
            const uint32_t t = 2u * (j - my_first), sl = t % PP_SLOTS;
            const bool mine = j >= my_lo && j < my_hi;
            const int i = j - my_lo;
            if (mine && !tbar_wait_warp(i == 0 ? &q_full[g] : &s_read[g], i == 0 ? 0u : (uint32_t)((i - 1) & 1), s_abort)) return false;
            if (!tbar_wait_warp(&full[sl], (t / PP_SLOTS) & 1u, s_abort)) return false;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one()) {
                if (mine) {
                    const uint64_t dk = dk0 + (uint64_t)((sl * PP_TILE) >> 4);
#pragma unroll
                    for (int k = 0; k < DH / 16; ++k)
                        umma_bf16(tmem_s, dq + (uint64_t)(((k >> 2) * ATOM_Q) >> 4) + 2 * (k & 3), dk + (uint64_t)(((k >> 2) * ATOM_KV) >> 4) + 2 * (k & 3),
                                  idesc_s, k > 0 ? 1u : 0u);
                    umma_commit(&s_full[g]);
                    tbar_arrive(&s_full[g]);
                    umma_commit(&empty[sl]);
                } else {
                    tbar_arrive(&empty[sl]);
                }
            }
            __syncwarp();
            return true;
        };
        ok = issue_s(my_first);
        for (int j = my_first; j < my_end && ok; ++j) {
            if (j + 1 < my_end && !issue_s(j + 1)) { ok = false; break; }
            const uint32_t t = 2u * (j - my_first) + 1, sl = t % PP_SLOTS;
            const bool mine = j >= my_lo && j < my_hi;
            const int i = j - my_lo;
            if (!tbar_wait_warp(&full[sl], (t / PP_SLOTS) & 1u, s_abort)) { ok = false; break; }
            if (mine && !tbar_wait_warp(&p_full[g * NP + i % NP], (uint32_t)((i / NP) & 1), s_abort)) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one()) {
                if (mine) {
                    const uint64_t dv = dv0 + (uint64_t)((sl * PP_TILE) >> 4);
                    const uint32_t p_at = tmem_p + (uint32_t)((i % NP) * (BK / 2));
#pragma unroll
                    for (int k = 0; k < BK / 16; ++k)               // 16 keys a step: 8 columns of P, 16 rows of V
                        pp_mma_ta(tmem_o, p_at + 8u * k, dv + (uint64_t)((k * 16 * 128) >> 4), idesc_o, (i > 0 || k > 0) ? 1u : 0u);
                    umma_commit(&o_full[g * NP + i % NP]);
                    umma_commit(&empty[sl]);
                } else {
                    tbar_arrive(&empty[sl]);
                }
            }
            __syncwarp();
        }
        if (!ok) atomicExch(s_abort, 1);
    } else {
        // ---- softmax warps: a lane of tensor memory is a query row; warps q and q + 4 of a group have a half of a block's keys each
        const int g = warp >> 3, q = warp & 3, half = (warp >> 2) & 1, r = q * 32 + lane;
        const int my_lo = GROUPS == 1 || g == 0 ? lo[0] : lo[GROUPS - 1], my_hi = GROUPS == 1 || g == 0 ? hi[0] : hi[GROUPS - 1], n_i = my_hi - my_lo;
        const int group_first = q_first + g * 128, q_pos = group_first + r;
        const int group_rows = n_rows - g * 128;                    // (may be none, or more than 128)
        const uint32_t lane_addr = (uint32_t)(q * 32) << 16;
        const uint32_t tmem_s = tmem + g * 256 + lane_addr, tmem_o = tmem_s + BK, tmem_p = tmem_o + DH;
        unsigned char* q_tile = q_tiles + g * Q_BYTES;
        float* sp = s_part + g * 256;
        const unsigned win_eff = window > 0 ? (unsigned)window : 0x7fffffffu;    // key visible: 0 ≤ q_pos − key < win_eff
        {
            // the queries, eight entries a piece, in the producers' order, as float16 divided by a power of two that takes the CTA's largest to 2^14: their
            // eight bits are all there but for numbers 2^-31 of that
            constexpr int PIECES = 128 * (DH / 8) / 256;
            uint4 v[PIECES];
            uint32_t top = 0;
#pragma unroll
            for (int x = 0; x < PIECES; ++x) {
                const int idx = x * 256 + (threadIdx.x & 255), rr = idx / (DH / 8), c = idx % (DH / 8);
                v[x] = make_uint4(0u, 0u, 0u, 0u);
                if (rr < group_rows) v[x] = *reinterpret_cast<const uint4*>(qkv + (size_t)(row0 + t_first + g * 128 + rr) * ld + q_off + (size_t)h * DH + c * 8);
            }
#pragma unroll
            for (int x = 0; x < PIECES; ++x) {
                const uint32_t w[4] = {v[x].x, v[x].y, v[x].z, v[x].w};
#pragma unroll
                for (int y = 0; y < 4; ++y) {                       // (what is not finite stays so whatever it is divided by)
                    const uint32_t a = w[y] & 0x7fffu, b = w[y] >> 16 & 0x7fffu;
                    top = max(top, max(a < 0x7f80u ? a : 0u, b < 0x7f80u ? b : 0u));
                }
            }
            top = __reduce_max_sync(0xffffffffu, top);
            if (lane == 0) {
                atomicMax(s_top, (int)top);
                tbar_arrive(q_known);
            }
            __syncwarp();
            if (n_i > 0 && tbar_wait_warp(q_known, 0, s_abort)) {
                const float down = pp_power(-pp_up((uint32_t)*s_top));
#pragma unroll
                for (int x = 0; x < PIECES; ++x) {
                    const int idx = x * 256 + (threadIdx.x & 255), rr = idx / (DH / 8), c = idx % (DH / 8);
                    const uint32_t w[4] = {v[x].x, v[x].y, v[x].z, v[x].w};
                    uint32_t o[4];
#pragma unroll
                    for (int y = 0; y < 4; ++y) {                   // entries (y, y + 4)
                        const uint32_t lo = w[y >> 1], hi = w[2 + (y >> 1)];
                        const __half2 two = (y & 1) ? __floats2half2_rn(__uint_as_float(lo & 0xffff0000u) * down, __uint_as_float(hi & 0xffff0000u) * down)
                                                    : __floats2half2_rn(__uint_as_float(lo << 16) * down, __uint_as_float(hi << 16) * down);
                        o[y] = *reinterpret_cast<const uint32_t*>(&two);
                    }
                    *reinterpret_cast<uint4*>(q_tile + (c >> 3) * ATOM_Q + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) tbar_arrive(&q_full[g]);
            }
        }
        float m_run = -INFINITY, l_run = 0.f;                       // the row's reference point; the sum of this half
        bool ok = true;
        auto wait_o = [&](int j) { return tbar_wait_warp(&o_full[g * NP + j % NP], (uint32_t)((j / NP) & 1), s_abort); };       // until O holds block j
        float unit = 0.f;                                           // (known once the first scores are there)
        // MASKED: some key of the block may be hidden from some row, and (is_far) some key or value may have a power of its own
        auto block = [&](int i, auto masked_c, bool there, uint32_t is_far) {
            constexpr bool MASKED = decltype(masked_c)::value;
            const int k0 = (my_lo + i) * BK + half * HK;            // the half's first key
            // chunks of 32 keys of which a row of this warp sees any (those behind lie above the diagonal)
            const int q_top = group_first + q * 32 + 31;
            const int n_live = MASKED ? (q_top < k0 ? 0 : min(NC, ((q_top - k0) >> 5) + 1)) : NC;
            // (a warp that has given up goes on meeting its neighbour, who may not have, until both have: with nothing to tell)
            if (!there) {
                ok = false;
                uint32_t any;
                asm volatile("{\n.reg .pred p, q;\nsetp.ne.b32 p, %1, 0;\nbarrier.cta.red.or.pred q, %2, 64, p;\nselp.u32 %0, 1, 0, q;\n}\n"
                             : "=r"(any) : "r"(0u), "r"(1 + g * 4 + q) : "memory");
                if (any) {
                    asm volatile("bar.sync %0, 64;" ::"r"(1 + g * 4 + q) : "memory");
                    asm volatile("bar.sync %0, 64;" ::"r"(1 + g * 4 + q) : "memory");
                }
                return;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t s_at = tmem_s + (uint32_t)(half * HK), p_at = tmem_p + (uint32_t)((i % NP) * (BK / 2) + half * (HK / 2));
            uint32_t sv[NC][32];
            unit = s_unit[0];
            const float2* far = s_far + ((my_lo + i - my_first) % PP_SLOTS) * 64;
            // Exponentials of a chunk, x times `by` being scores in units of log2(e), against m_use and 2^PP_UP times; P as float16 into tensor memory, their
            // sum onto `sum`.
            auto chunk = [&](int c, const uint32_t (&x)[32], float by, float m_use, uint64_t (&sum)[2]) {
                uint32_t pk[16];
                const int d0 = q_pos - (k0 + c * 32);               // q_pos − key for e = 0
                const uint64_t by2 = pp_two(by, by), from = pp_two(PP_UP - m_use, PP_UP - m_use);
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    float p0, p1;
                    pp_apart(pp_fma2(pp_two(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), by2, from), p0, p1);
                    p0 = pp_exp2(p0);
                    p1 = pp_exp2(p1);
                    if (MASKED) {
                        p0 = (unsigned)(d0 - e) < win_eff ? p0 : 0.f;
                        p1 = (unsigned)(d0 - e - 1) < win_eff ? p1 : 0.f;
                    }
                    sum[(e >> 1) & 1] = pp_add2(sum[(e >> 1) & 1], pp_two(p0, p1));
                    const __half2 two = __floats2half2_rn(p0, p1);
                    pk[e >> 1] = *reinterpret_cast<const uint32_t*>(&two);
                }
                pp_st16(p_at + (uint32_t)(c * 16), pk);
            };
            // a chunk's scores with the powers of its keys and values; with m_use, returns the sum of its weights without those of the values
            auto with_powers = [&](int c, uint32_t (&x)[32], float m_use) {
                float plain = 0.f;
                const int d0 = q_pos - (k0 + c * 32);
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const int key = half * HK + c * 32 + e;
                    const float2 power = (is_far >> (key / (BK / NPROD) * 8) & 255u) != 0u ? far[key] : make_float2(1.f, 0.f);
                    const float score = __uint_as_float(x[e]) * power.x * unit;
                    plain += (unsigned)(d0 - e) < win_eff ? pp_exp2(score + (PP_UP - m_use)) : 0.f;
                    x[e] = __float_as_uint(score + power.y);
                }
                return plain;
            };
            auto total = [](const uint64_t (&sum)[2]) {
                float a0, a1, b0, b1;
                pp_apart(sum[0], a0, a1);
                pp_apart(sum[1], b0, b1);
                return (a0 + a1) + (b0 + b1);
            };
            // whether any row of the two warps asks for it
            auto either = [&](bool mine) {
                uint32_t any;
                asm volatile("{\n.reg .pred p, q;\nsetp.ne.b32 p, %1, 0;\nbarrier.cta.red.or.pred q, %2, 64, p;\nselp.u32 %0, 1, 0, q;\n}\n"
                             : "=r"(any) : "r"((uint32_t)mine), "r"(1 + g * 4 + q) : "memory");
                return any != 0;
            };
            // The weights' reference point m_run moves to the row's maximum where that lies 2^least above it (both halves' maxima meet in shared memory);
            // returns what the sums so far are to be multiplied by.
            auto move_reference = [&](float m_half, float least) {
                sp[half * 128 + r] = m_half;
                asm volatile("bar.sync %0, 64;" ::"r"(1 + g * 4 + q) : "memory");
                const float m_blk = fmaxf(m_half, sp[(half ^ 1) * 128 + r]);
                const float m_new = m_blk > m_run + least ? m_blk : m_run;
                const float corr = m_run == -INFINITY ? 1.f : pp_exp2(m_run - m_new);    // (from −inf on the row's sums are 0 so far)
                l_run *= corr;
                m_run = m_new;
                asm volatile("bar.sync %0, 64;" ::"r"(1 + g * 4 + q) : "memory");        // (read, before the next is written)
                return corr;
            };
            auto reference = [&]() { return m_run == -INFINITY ? 0.f : m_run; };         // (a row that sees nothing yet: every weight is 0)
            float corr = 1.f, sum = 0.f;
            bool moved;
            // (P goes where the product of NP blocks before has read it; where O is to be scaled, all blocks before are in it)
            if (!MASKED) {
#pragma unroll
                for (int c = 0; c < NC; ++c) tmem_ld32(s_at + 32u * c, sv[c]);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) tbar_arrive(&s_read[g]);
                // No maximum is looked for while the weights against the reference point stay small: they are as exact in float16 up to 2^15 as up to
                // 1.  A row whose weights of this block add up to more (for random rows hardly any behind the first block) moves its reference
                // point, and the two warps begin the block anew.
                if (i > 0) {
                    if (i >= NP && !wait_o(i - NP)) ok = false;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    uint64_t s2[2] = {0ull, 0ull};
#pragma unroll
                    for (int c = 0; c < NC; ++c) chunk(c, sv[c], unit, reference(), s2);
                    sum = total(s2);
                }
                moved = either(i == 0 || m_run == -INFINITY || sum > PP_MOST);
                if (moved) {
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int x = 0; x < 32; ++x) mx[x & 3] = fmaxf(mx[x & 3], __uint_as_float(sv[c][x]) * unit);
                    corr = move_reference(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), PP_LEAST);
                    if (i > 0 && !wait_o(i - 1)) ok = false;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    uint64_t s2[2] = {0ull, 0ull};
#pragma unroll
                    for (int c = 0; c < NC; ++c) chunk(c, sv[c], unit, reference(), s2);
                    sum = total(s2);
                }
                if (!ok) return;
            } else {
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                for (int c = 0; c < n_live; ++c) {
                    tmem_ld32(s_at + (uint32_t)(c * 32), sv[0]);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (is_far != 0u) with_powers(c, sv[0], 0.f);
                    const float by = is_far != 0u ? 1.f : unit;
                    const int d0 = q_pos - (k0 + c * 32);
#pragma unroll
                    for (int x = 0; x < 32; ++x) mx[x & 3] = fmaxf(mx[x & 3], (unsigned)(d0 - x) < win_eff ? __uint_as_float(sv[0][x]) * by : -INFINITY);
                }
                const float m_half = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                moved = either(m_half > m_run + PP_LEAST);
                if (moved) corr = move_reference(m_half, PP_LEAST);
                const int before = moved ? i - 1 : i - NP;
                if (before >= 0) {
                    if (!wait_o(before)) { ok = false; return; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                }
                uint64_t s2[2] = {0ull, 0ull};
                float plain = 0.f;
#pragma unroll 1
                for (int c = 0; c < NC; ++c) {
                    if (c < n_live) {
                        tmem_ld32(s_at + (uint32_t)(c * 32), sv[0]);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        if (is_far != 0u) plain += with_powers(c, sv[0], reference());
                        chunk(c, sv[0], is_far != 0u ? 1.f : unit, reference(), s2);
                    } else {
                        uint32_t none[16];
#pragma unroll
                        for (int x = 0; x < 16; ++x) none[x] = 0u;
                        pp_st16(p_at + (uint32_t)(c * 16), none);
                    }
                }
                sum = is_far != 0u ? plain : total(s2);
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) tbar_arrive(&s_read[g]);
            }
            l_run += sum;
            if (i > 0 && moved) {                                           // a row's reference point moved: its O (a half of the columns here) follows
#pragma unroll
                for (int d0 = 0; d0 < HD; d0 += 32) {
                    uint32_t ov[32];
                    tmem_ld32(tmem_o + (uint32_t)(half * HD + d0), ov);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int x = 0; x < 32; ++x) ov[x] = __float_as_uint(__uint_as_float(ov[x]) * corr);
                    pp_st32(tmem_o + (uint32_t)(half * HD + d0), ov);
                }
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) tbar_arrive(&p_full[g * NP + i % NP]);
        };
        for (int i = 0; i < n_i; ++i) {                             // (uniform over the group)
            const bool there = ok && tbar_wait_warp(&s_full[g], (uint32_t)(i & 1), s_abort);
            const uint32_t is_far = there ? s_any_far[(my_lo + i - my_first) % PP_SLOTS] : 0u;
            if (is_far != 0u || window > 0 || (my_lo + i) * BK + BK - 1 > group_first) block(i, std::true_type{}, there, is_far);
            else block(i, std::false_type{}, there, 0u);
        }
        // the row's result, a half of the columns a thread and 32 of them at a time, and the sum of both halves of the keys
        const bool any_o = n_i > 0 && ok && wait_o(n_i - 1);
        if (n_i > 0 && !any_o) {
            ok = false;
            atomicExch(s_abort, 1);
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        auto result = [&](int d0, float (&o)[32]) {
            uint32_t ov[32];
            if (any_o) {
                tmem_ld32(tmem_o + (uint32_t)(half * HD + d0), ov);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            }
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = any_o ? __uint_as_float(ov[x]) * s_unit[1] : 0.f;
        };
        // as bfloat16, entries in order again, into shared memory (Q's tile: no MMA reads it any more)
        auto leave = [&](int d0, const float (&o)[32], float inv) {
#pragma unroll
            for (int d = 0; d < 32; d += 8) {
                uint4 pk;
                pk.x = pack2(o[d] * inv, o[d + 2] * inv); pk.y = pack2(o[d + 4] * inv, o[d + 6] * inv);
                pk.z = pack2(o[d + 1] * inv, o[d + 3] * inv); pk.w = pack2(o[d + 5] * inv, o[d + 7] * inv);
                const int c = (half * HD + d0 + d) >> 3;
                *reinterpret_cast<uint4*>(q_tile + (c >> 3) * ATOM_Q + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = pk;
            }
        };
        auto inverse = [&]() { return m_run == -INFINITY && l_run == 0.f ? 0.f : 1.f / l_run; };     // (values 2^126 apart: infinite rather than 0)
        asm volatile("bar.sync %0, 256;" ::"r"(9 + g) : "memory");  // (also behind the last block's maxima)
        sp[half * 128 + r] = l_run;
        asm volatile("bar.sync %0, 256;" ::"r"(9 + g) : "memory");
        l_run = sp[r] + sp[128 + r];
        bool writes_out = group_rows > 0;
        if (tile_parts == 1) {
            const float inv = inverse();
#pragma unroll 1
            for (int d0 = 0; d0 < HD; d0 += 32) {
                float o[32];
                result(d0, o);
                leave(d0, o, inv);
            }
        } else if (group_rows > 0) {
            // leave this part's result in scratch ([d][row], so that a warp writes whole lines), then see whether the tile's other
            // parts are all there
            const size_t tile_id = ((size_t)*s_place * H + h) * GROUPS + g;
            const float* parts = partials + tile_id * n_parts * pp_part_floats(DH);
            float* mine = partials + (tile_id * n_parts + part) * pp_part_floats(DH);
#pragma unroll 1
            for (int d0 = 0; d0 < HD; d0 += 32) {
                float o[32];
                result(d0, o);
#pragma unroll
                for (int x = 0; x < 32; ++x) mine[(half * HD + d0 + x) * 128 + r] = o[x];
            }
            if (half == 0) {
                mine[DH * 128 + r] = m_run;
                mine[DH * 128 + 128 + r] = l_run;
            }
            __threadfence();
            asm volatile("bar.sync %0, 256;" ::"r"(9 + g) : "memory");
            if ((threadIdx.x & 255) == 0) {
                const int before = atomicAdd(&counters[tile_id], 1);
                s_last[g] = (before == tile_parts - 1) ? 1 : 0;
                if (before == tile_parts - 1) counters[tile_id] = 0;             // left as it was found
            }
            asm volatile("bar.sync %0, 256;" ::"r"(9 + g) : "memory");
            writes_out = s_last[g] != 0;
            if (writes_out) {
                __threadfence();
                // every part in turn, this CTA's own included: the sum does not depend on who came last
                m_run = -INFINITY;
                for (int pt = 0; pt < tile_parts; ++pt) m_run = fmaxf(m_run, __ldcg(parts + pt * pp_part_floats(DH) + DH * 128 + r));
                auto weight = [&](int pt) {                         // (sums that are not numbers stay so)
                    const float m_p = __ldcg(parts + pt * pp_part_floats(DH) + DH * 128 + r);
                    return m_p == -INFINITY ? 0.f : pp_exp2(m_p - m_run);
                };
                l_run = 0.f;
                for (int pt = 0; pt < tile_parts; ++pt) l_run = fmaf(__ldcg(parts + pt * pp_part_floats(DH) + DH * 128 + 128 + r), weight(pt), l_run);
                const float inv = inverse();
#pragma unroll 1
                for (int d0 = 0; d0 < HD; d0 += 32) {
                    float o[32];
#pragma unroll
                    for (int x = 0; x < 32; ++x) o[x] = 0.f;
#pragma unroll 1
                    for (int pt = 0; pt < tile_parts; ++pt) {
                        const float* theirs = parts + pt * pp_part_floats(DH) + (half * HD + d0) * 128 + r;
                        const float w = weight(pt);
                        float v[32];
#pragma unroll
                        for (int x = 0; x < 32; ++x) v[x] = __ldcg(theirs + x * 128);
#pragma unroll
                        for (int x = 0; x < 32; ++x) o[x] = fmaf(v[x], w, o[x]);
                    }
                    leave(d0, o, inv);
                }
            }
        }
        if (writes_out) {
            // each warp writes whole rows, so that a store instruction fills whole lines
            asm volatile("bar.sync %0, 64;" ::"r"(1 + g * 4 + q) : "memory");
            if (ok) {
                constexpr int PIECES = DH / 8, AT_ONCE = 32 / PIECES;
#pragma unroll
                for (int it = 0; it < 16 / AT_ONCE; ++it) {
                    const int rr = q * 32 + half * 16 + it * AT_ONCE + lane / PIECES, c = lane % PIECES;
                    if (rr < group_rows) {
                        const uint4 pk = *reinterpret_cast<const uint4*>(q_tile + (c >> 3) * ATOM_Q + rr * 128 + (((c & 7) ^ (rr & 7)) << 4));
                        *reinterpret_cast<uint4*>(out + (size_t)(row0 + t_first + g * 128 + rr) * ld_out + (size_t)h * DH + c * 8) = pk;
                    }
                }
            }
        }
    }
    pdl_launch_dependents();                                        // (CTAs of the next kernel taken in earlier would sit on the places that are free then)
    // everyone meets here on every path; then the allocating warp gives the tensor memory back
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (*s_abort) {                                                 // MMAs under way read this CTA's shared memory: wait for them (bounded)
        if (warp >= SOFT + NPROD) {
            if (elect_one()) umma_commit(drained);
            __syncwarp();
            tbar_wait_warp(drained, 0, s_never);
        }
        __syncthreads();
    }
    if (warp == SOFT) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    if (threadIdx.x == 0 && *s_abort) atomicOr(dev_err, VLRF_DEVERR_WAIT_TIMEOUT);
}

template <int DH, int GROUPS>
int pp_launch(const void* qkv, int ld, int q_off, const void* Kq, const void* Kp, const void* Vq, const void* Vp, int n_blocks, const int* block_table,
              int max_blocks, const int* seq_slot, const int* seq_start, const int* seq_pos0, void* out, int ld_out, int n_tokens, int n_seqs, int max_new, int H,
              int Hkv, float scale, int window, int least_new, int n_parts, int part_blocks, int n_places, float* partials, int* counters, int* dev_err,
              cudaStream_t stream) {
    const size_t smem = 1024 + (size_t)GROUPS * 128 * DH * 2 + (size_t)PP_RING + GROUPS * 256 * 4 + (PP_RING / (PP_BK * DH * 2)) * (64 * 8 + 4) + 48 * 8;
    static DeviceMarks marks;
    auto kern = attn_packed_prefill_kernel<DH, GROUPS>;
    cudaError_t e = allow_shared_memory(marks, kern, smem);
    if (e != cudaSuccess) return vlrf_fail(VLRF_ERR_CUDA, "attn_packed_prefill: %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    const long long tiles = (max_new + GROUPS * 128 - 1) / (GROUPS * 128);
    // A place a tile that there can be (⌈len / rows⌉ over the sequences), where that is less than half of the longest sequence's tiles for every sequence: a
    // CTA that finds nothing to do takes an SM's place for a microsecond, and one that looks its tile up starts half a microsecond later
    // (five sequences of 1 to 640 tokens, 25 heads of 64, window 256: 25.4 us, so 24.0).
    const long long flat = n_tokens / (GROUPS * 128) + n_seqs;
    const bool use_flat = 2 * flat < tiles * n_seqs && flat * n_parts <= 65535;
    VLRF_REQUIRE(use_flat || tiles * n_parts <= 65535, "attn_packed_prefill: %lld tiles of %d parts are too many for one launch", tiles, n_parts);
    const dim3 grid(H, use_flat ? 1 : n_seqs, (unsigned)((use_flat ? flat : tiles) * n_parts));
    e = launch_chained(kern, grid, dim3(pp_threads(GROUPS)), smem, stream, (const __nv_bfloat16*)qkv, ld, q_off,
                       (const unsigned char*)Kq, (const uint32_t*)Kp, (const unsigned char*)Vq, (const uint32_t*)Vp, n_blocks, block_table, max_blocks, seq_slot,
                       seq_start, seq_pos0, (__nv_bfloat16*)out, ld_out, H, Hkv, scale, window, n_parts, part_blocks, partials, counters, (int)tiles, n_seqs,
                       use_flat ? (int)flat : 0, n_places, least_new, dev_err);
    if (e != cudaSuccess) return vlrf_fail(VLRF_ERR_CUDA, "attn_packed_prefill: %s", cudaGetErrorString(e));
    return vlrf_check_launch("attn_packed_prefill");
}
}  // namespace

extern "C" int vlrf_attn_packed_prefill_takes(int H, int Hkv, int dh, int BT, int ld, int q_off, int ld_out) {
    return H > 0 && Hkv > 0 && H % Hkv == 0 && (dh == 64 || dh == 128) && BT == PP_CB && ld % 8 == 0 && q_off % 8 == 0 && ld_out % 8 == 0;
}
extern "C" int vlrf_attn_packed_prefill_max_parts() { return PP_MAX_PARTS; }

// Scratch of a launch with n_parts > 1: float32 numbers of partials, int32 numbers of counters.
extern "C" int vlrf_attn_packed_prefill_scratch(int n_seqs, int max_new, int H, int dh, int groups, int n_parts, long long* floats, long long* ints) {
    VLRF_REQUIRE(n_seqs >= 0 && max_new >= 0 && H > 0 && (dh == 64 || dh == 128) && (groups == 1 || groups == 2) && n_parts >= 1, "attn_packed_prefill: bad sizes");
    const long long tiles = (long long)((max_new + groups * 128 - 1) / (groups * 128)) * groups * n_seqs * H;
    *floats = n_parts > 1 ? tiles * n_parts * pp_part_floats(dh) : 0;
    *ints = n_parts > 1 ? tiles : 0;
    return VLRF_OK;
}

// With scratch for n_places tiles (of a head): n_places · H · groups · n_parts · (128 dh + 256) float32 numbers, n_places · H · groups int32 numbers.
extern "C" int vlrf_attn_packed_prefill_places(const void* qkv, int ld, int q_off, const void* Kq, const void* Kp, const void* Vq, const void* Vp, int n_blocks,
                                               const int* block_table, int max_blocks, const int* seq_slot, const int* seq_start, const int* seq_pos0,
                                               void* out, int ld_out, int n_tokens, int n_seqs, int max_new, int H, int Hkv, int dh, int BT, float scale,
                                               int window, int least_new, int groups, int n_parts, int part_blocks, int n_places, float* partials,
                                               int* counters, int* dev_err, cudaStream_t stream) {
    VLRF_REQUIRE(vlrf_attn_packed_prefill_takes(H, Hkv, dh, BT, ld, q_off, ld_out),
                 "attn_packed_prefill: %d heads over %d of %d, blocks of %d, row strides %d and %d are not taken", H, Hkv, dh, BT, ld, ld_out);
    VLRF_REQUIRE(n_tokens >= 0 && n_seqs >= 0 && n_seqs <= 65535 && max_new >= 0 && max_blocks > 0 && n_blocks >= 0 && window >= 0 && least_new >= 1 &&
                     dev_err != nullptr,
                 "attn_packed_prefill: bad arguments");
    VLRF_REQUIRE(scale >= 0.f, "attn_packed_prefill: a scale of %g is negative", (double)scale);       // (a row's maximum is taken of the raw scores)
    VLRF_REQUIRE(groups == 1 || groups == 2, "attn_packed_prefill: %d groups of 128 queries a CTA (1 or 2)", groups);
    VLRF_REQUIRE(n_parts >= 1 && n_parts <= PP_MAX_PARTS && part_blocks >= 1 && (n_parts == 1 || (partials != nullptr && counters != nullptr)),
                 "attn_packed_prefill: %d parts (1 to %d; more than one wants scratch)", n_parts, PP_MAX_PARTS);
    VLRF_REQUIRE(n_places >= 0, "attn_packed_prefill: scratch for %d tiles", n_places);
    for (const void* p : {qkv, Kq, Kp, Vq, Vp, (const void*)out})
        VLRF_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15) == 0, "attn_packed_prefill: tensors begin on 16 bytes");
    if (n_seqs == 0 || max_new == 0) return VLRF_OK;
#define GO(DH, G) pp_launch<DH, G>(qkv, ld, q_off, Kq, Kp, Vq, Vp, n_blocks, block_table, max_blocks, seq_slot, seq_start, seq_pos0, out, ld_out, n_tokens, \
                                   n_seqs, max_new, H, Hkv, scale, window, least_new, n_parts, part_blocks, n_places, partials, counters, dev_err, stream)
    if (dh == 64) return groups == 1 ? GO(64, 1) : GO(64, 2);
    return groups == 1 ? GO(128, 1) : GO(128, 2);
#undef GO
}

// With scratch for every tile that the sequences may have (vlrf_attn_packed_prefill_scratch).
extern "C" int vlrf_attn_packed_prefill(const void* qkv, int ld, int q_off, const void* Kq, const void* Kp, const void* Vq, const void* Vp, int n_blocks,
                                        const int* block_table, int max_blocks, const int* seq_slot, const int* seq_start, const int* seq_pos0, void* out,
                                        int ld_out, int n_tokens, int n_seqs, int max_new, int H, int Hkv, int dh, int BT, float scale, int window, int least_new,
                                        int groups, int n_parts, int part_blocks, float* partials, int* counters, int* dev_err, cudaStream_t stream) {
    VLRF_REQUIRE(groups == 1 || groups == 2, "attn_packed_prefill: %d groups of 128 queries a CTA (1 or 2)", groups);
    const long long tiles = (long long)max(n_seqs, 0) * ((max(max_new, 0) + groups * 128ll - 1) / (groups * 128));
    return vlrf_attn_packed_prefill_places(qkv, ld, q_off, Kq, Kp, Vq, Vp, n_blocks, block_table, max_blocks, seq_slot, seq_start, seq_pos0, out, ld_out, n_tokens,
                                           n_seqs, max_new, H, Hkv, dh, BT, scale, window, least_new, groups, n_parts, part_blocks,
                                           (int)min(tiles, 0x7fffffffll), partials, counters, dev_err, stream);
}
