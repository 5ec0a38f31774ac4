// Attention over the 4-bit key/value cache (format: kv4.cu).
//
// With k'_t = m_t + s_t c_t for the key at position t (and v'_t alike for the value),
//     score_t = (q . k'_t) / sqrt(head) = (s_t (q . c_t) + m_t sum q) / sqrt(head)
//     out = sum_t p_t (s_t c_t + m_t),  p = softmax over positions 0 .. the row's own,
// so the products with codes are whole-number products, and s and m enter per position only.
//
// Tensor-core products without unpacking. A 4-bit code masked out of a 16-bit half, at bits 0-3
// or 4-7, is the fp16 subnormal c 2^-24 or 16 c 2^-24: one AND makes two exact operands of
// mma.m16n8k16, and the powers of two are undone in the query (K) and the output (V). The unit
// aligns products by their exponent fields, so subnormals lose low bits of a long factor; the
// other operand is therefore a whole number of at most 11 bits, whose products and sums are exact
// (with an fp16 value there, f32 results were 7e-5 off instead of some 1e-7). The cache
// is the 16-row operand (16 positions for K, 16 dims for V), read once for up to eight query heads
// of its group (more are units of their own); the queries and the weights are the 8-column one, each head taking two columns of
// fp16, the whole number and the rest, together 22 bits. So f32 results keep their digits, and one
// lane's accumulators all belong to one head: its maximum, sum and rescaling need no exchange.
//
// Bound: latency. A warp's 32 positions (head 128) are 4352 bytes and about 490 instructions, 32 of
// them mma. Each warp keeps the next 32 positions on their way into shared memory while it computes
// on the present ones; registers and shared memory hold 16 warps an SM. Measured (8 kv heads of 4
// query heads, head 128): one row of 131072 positions 36.9 us (143 MB, 3.9 TB/s, half the issue
// slots and 0.6 of the memory's rate used: too few bytes under way, and barriers at the ends); 64
// rows of 1 to 8192, 56.5 us (265 MB, 4.7 TB/s); one of 8001, 10.2 us. 256 rows of 1 to 1024
// positions of 12 heads of 64 take 44 us (113 MB, 2.6 TB/s): five units a block, whose starts and
// joins are what its barriers wait for.
//
// Split: the tiles (a turn of all warps of a block) of all units (a row's or a slot block's
// positions of one kv head) form one line that the blocks of one wave share equally, so rows of
// unlike lengths and few rows of great length fill the device alike. A unit that several blocks
// meet is joined by the last of them to finish, in line order: results do not depend on which
// that is. Where units are more than blocks, each counts kLead tiles more than it has, about what
// starting and joining it takes (counted by tiles alone, blocks of short units finished last).
#include <cuda_fp16.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "kv4.h"
#include "tma.cuh"  // smem_u32

namespace ab {

namespace {

// Warps of an SM, in two blocks of eight (NW below) or, for units that outnumber the small blocks,
// four of four: units start and end without the other blocks' waiting. Eight warps against four,
// own caches of rows of 1 to so many positions, 32 heads of 8 kv heads, head 128, bf16: 512 rows of
// 200 54 us against 40, 256 of 1000 53 against 45, 128 of 4000 64 against 58, but 64 of 8192 (512
// units) 56 against 60, one of 131072 36 against 41 (f32): with long stretches there are twice the
// parts to join. Of eight slots a unit at head 97 to 128 only three small blocks fit an SM's shared
// memory: 256 rows of 2000, 64 heads of 8, 107 us against 131, so it is eight warps there. A third
// block of eight (80 registers) measured 43 us where two took 37 at one row of 128k positions; one
// of 16 warps 37, and 101 where two took 73 at 256 rows of 12 heads.
constexpr int kSmWarps = 16;
constexpr uint32_t kTurn = 32;  // positions of one warp's turn; a tile is one of a block's warps
// Tiles that a unit is taken to cost beyond its own. Eight warps: 0, 1, 2, 3 and 8 measured 69.5,
// 59.1, 56.4, 57.7 and 62.5 us at 64 ragged rows of up to 8192 positions (as above). Four: 2, 3
// and 4 measured 43.7, 42.9 and 43.3 at 256 of up to 1024 (12 heads, head 64, f32).
template <int NW>
constexpr uint32_t kLead = NW == 8 ? 2 : 3;
// More query slots than these of a kv head over one cache go to tcgen05 (bf16 outputs; here against
// there, 8 kv heads, head 128): 64 slots of 2048 positions 15 us against 24, 256 of 64 positions 9
// against 14 and of 2000 32 against 26, 512 of 128 15 against 14, 2048 of 1024 89 against 33.
constexpr uint64_t kTensorSlots = 256;
constexpr float kLog2e = 1.4426950408889634f;

struct Kv4AttnParams {
    const float* q;  // [rows, heads, head]
    void* out;       // [rows, heads * head]
    Kv4View c;
    uint32_t rows, heads, group;
    uint32_t items;     // rows with a cache each, or blocks of query slots over one cache
    uint32_t per_item;  // kv heads x slot blocks of a row's group
    int shared;         // rows share one cache
    uint32_t lead;      // tiles that a unit counts more than it has
    int qvec, ovec;     // 16-byte loads of q, four outputs at once
    float* part;        // [2 grid][slots][32 W + 2] partial results
    uint32_t* tickets;  // [items * per_item], zero between launches
    const Step* step;
    uint32_t* flags;
};

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same from zero.
__device__ __forceinline__ void mma16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// 8 x 8 transpose of 16-bit elements held two a lane (row lane / 4, columns 2 (lane % 4) ..).
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// Reads of the cache: not the non-coherent path, the writer may be the grid before this one.
__device__ __forceinline__ uint4 ld16(const void* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p));
    return r;
}
__device__ __forceinline__ uint32_t ld4(const void* p) {
    uint32_t r;
    asm volatile("ld.global.u32 %0, [%1];" : "=r"(r) : "l"(p));
    return r;
}
// ---- a turn's rows in shared memory ---------------------------------------------------------
// [32 rows of K codes][32 rows of V codes][K scales][V scales]. The 16-byte chunks of a row are
// permuted by its number, so that eight consecutive rows of one chunk, which is what the lanes
// read at a time, are in unlike banks (rows of 16 and 48 bytes are so by themselves).
template <int W>
struct Stage {
    static constexpr uint32_t ROW = 16 * W;
    static constexpr uint32_t V = kTurn * ROW, KS = 2 * V, VS = KS + 4 * kTurn;
    static constexpr uint32_t BYTES = VS + 4 * kTurn;
    __device__ __forceinline__ static uint32_t place(uint32_t row, uint32_t chunk) {
        if constexpr (W == 4) chunk ^= row >> 1 & 3;
        if constexpr (W == 2) chunk ^= row >> 2 & 1;
        return row * ROW + chunk * 16;
    }
};
constexpr uint32_t kStages = 2;

// Asynchronous copies; those past the last row (size 0) write zeros and read nothing.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t size) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size)
                 : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, uint32_t size) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(size)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() {
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint32_t lds4(uint32_t at) {
    uint32_t x;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
    return x;
}
// A lane's quarter of a K row: W words.
template <int W>
__device__ __forceinline__ void load_k(uint32_t at, uint32_t (&w)[W]) {
    if constexpr (W == 4) {
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(at)
                     : "memory");
    } else if constexpr (W == 2) {
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                     : "=r"(w[0]), "=r"(w[1])
                     : "r"(at)
                     : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < W; i++) w[i] = lds4(at + 4 * i);
    }
}
// One chunk (eight units of four codes) of all 32 V rows, transposed: y[b] holds unit r of the
// rows 8 b + 2 c (low half) and 8 b + 2 c + 1. `at`: the chunk of row `lane`.
__device__ __forceinline__ void load_v(uint32_t at, uint32_t (&y)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(y[0]), "=r"(y[1]), "=r"(y[2]), "=r"(y[3])
                 : "r"(at)
                 : "memory");
}

// Positions that the rows of item i attend over.
template <uint32_t S>
__device__ __forceinline__ uint32_t item_length(const Kv4AttnParams& p, uint32_t i) {
    uint32_t r0 = i, r1 = i;
    if (p.shared) {
        r0 = i * S / p.group;
        r1 = min(p.rows - 1, (i * S + S - 1) / p.group);
    }
    uint32_t n = 0;
    for (uint32_t r = r0; r <= r1; r++) {
        const uint32_t pos = p.step[r].position;
        if (pos < p.c.seq) n = max(n, pos + 1);
    }
    return n;
}
// Tiles of the line; at least one, so that a row without positions is written too.
template <int NW>
__device__ __forceinline__ uint32_t tiles_of(uint32_t length) {
    return max(1u, (length + NW * kTurn - 1) / (NW * kTurn));
}

// The line of `total` tiles over `blocks` blocks: the first `more` of them take one tile more.
struct Line {
    uint32_t blocks = 0, each = 0, more = 0;
    __device__ __forceinline__ Line() {}
    __device__ __forceinline__ Line(uint32_t total, uint32_t most) {
        blocks = min(total, most);
        each = total / blocks;
        more = total % blocks;
    }
    __device__ __forceinline__ uint32_t begin(uint32_t block) const {
        return block * each + min(block, more);
    }
    __device__ __forceinline__ uint32_t block_of(uint32_t tile) const {
        const uint32_t cut = more * (each + 1);
        return tile < cut ? tile / (each + 1) : more + (tile - cut) / each;
    }
};

// What a block's first warp finds for all: a unit (tiles [at, until) of the line) and the
// positions of it that are the block's.
struct Span {
    uint32_t item, nth, kvh, sub, at, until, t_begin, t_end;
};

// A unit whose parts, those of blocks first .. first + parts - 1, are to be joined.
struct Job {
    uint32_t item, kvh, sub, first, parts;
};

// One query of a unit: what its products with codes are scaled by, its sum, -8 times the sums of
// its two columns, the last position it attends over.
struct Slot {
    float scale, sum, first, rest;
    int32_t limit;
};

// One unit: S query slots over the positions of one kv head of one cache.
template <int W, uint32_t S, typename OT>
struct Unit {
    const Kv4AttnParams& p;
    uint32_t item, kvh, sub;
    // slot -> query row, head; false past the last
    __device__ __forceinline__ bool slot(uint32_t s, uint32_t* row, uint32_t* head) const {
        if (p.shared) {
            const uint32_t k = item * S + s;
            *row = k / p.group;
            *head = kvh * p.group + k % p.group;
            return *row < p.rows;
        }
        *row = item;
        *head = kvh * p.group + sub * S + s;
        return sub * S + s < p.group;
    }
    // Four dims from element 4 i of [S][32 W] on: x over the sum L (no positions: zeros).
    __device__ __forceinline__ void write(uint32_t i, const float4& x, float L) const {
        const uint32_t s = i / (8 * W), d = i % (8 * W) * 4, hd = p.c.head;
        uint32_t row, head;
        if (!slot(s, &row, &head) || d >= hd) return;
        OT* dst = (OT*)p.out + ((uint64_t)row * p.heads + head) * hd + d;
        const float f = L == 0.0f ? 0.0f : 1.0f / L;
        const float v[4] = {x.x * f, x.y * f, x.z * f, x.w * f};
        if (p.ovec) {
            if constexpr (sizeof(OT) == 4) {
                *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
                const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]),
                                     b = __floats2bfloat162_rn(v[2], v[3]);
                *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&a),
                                                            *reinterpret_cast<const uint32_t*>(&b));
            }
        } else {
#pragma unroll
            for (uint32_t k = 0; k < 4; k++)
                if (d + k < hd) dst[k] = from_f32<OT>(v[k]);
        }
    }
};

// Joins the parts of blocks first .. first + n - 1 in that order and writes the unit's rows.
// The [S][32 W] outputs are COLS groups of four; JG threads share one and take every JG-th part
// (what is left of the threads rests). A thread joins its parts as an online softmax does, so
// that weights and values are read in one round, AHEAD parts at a time. so, sm, sl: the block's
// shared arrays, free by now.
template <int W, int NW, uint32_t S, typename OT>
__device__ __forceinline__ void join_parts(const Unit<W, S, OT>& unit, uint32_t first, uint32_t n,
                                        uint32_t tid, float* so, float (*sm)[S],
                                           float (*sl)[S]) {
    constexpr uint32_t PART = S * (32 * W + 2), COLS = S * 8 * W;
    constexpr uint32_t THREADS = NW * 32, JG = COLS < THREADS ? THREADS / COLS : 1;
    static_assert(JG <= NW, "exchanged values fit where the warps' parts were");
    constexpr uint32_t AHEAD = 8;
#pragma unroll 1
    for (uint32_t c0 = 0; c0 < COLS; c0 += THREADS) {  // once, but with few threads
        const uint32_t col = COLS < THREADS ? tid % COLS : c0 + tid;
        const uint32_t jg = COLS < THREADS ? tid / COLS : (col < COLS ? 0 : 1);
        const uint32_t s = col / (8 * W);
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float J = -INFINITY, L = 0.0f;
        auto join = [&](const float4& v, float mj, float lj) {
            if (mj == -INFINITY) return;
            const float to = fmaxf(J, mj), a = ex2(J - to), b = ex2(mj - to);
            x.x = fmaf(v.x, b, x.x * a);
            x.y = fmaf(v.y, b, x.y * a);
            x.z = fmaf(v.z, b, x.z * a);
            x.w = fmaf(v.w, b, x.w * a);
            L = fmaf(lj, b, L * a);
            J = to;
        };
        for (uint32_t j0 = jg < JG ? jg : n; j0 < n; j0 += AHEAD * JG) {
            float4 v[AHEAD];
            float mj[AHEAD], lj[AHEAD];
#pragma unroll
            for (uint32_t u = 0; u < AHEAD; u++) {
                const uint32_t j = j0 + u * JG;
                // the unit begins inside the first block's stretch and before the others'
                const float* pj = unit.p.part + ((uint64_t)2 * (first + j) + (j == 0)) * PART;
                mj[u] = -INFINITY;
                if (j < n) {
                    mj[u] = __ldcg(pj + COLS * 4 + s);
                    lj[u] = __ldcg(pj + COLS * 4 + S + s);
                    v[u] = __ldcg(reinterpret_cast<const float4*>(pj) + col);
                }
            }
#pragma unroll
            for (uint32_t u = 0; u < AHEAD; u++) join(v[u], mj[u], lj[u]);
        }
        if constexpr (JG > 1) {
            if (jg < JG) {
                reinterpret_cast<float4*>(so)[jg * COLS + col] = x;
                sm[jg][s] = J;  // the same from every thread of a slot
                sl[jg][s] = L;
            }
            __syncthreads();
            if (jg == 0) {
#pragma unroll
                for (uint32_t g = 1; g < JG; g++)
                    join(reinterpret_cast<const float4*>(so)[g * COLS + col], sm[g][s], sl[g][s]);
            }
        }
        if (jg == 0) unit.write(col, x, L);
    }
}

// W: words of codes in a quarter row (head up to 32 W). NT: four query slots each. NW: warps.
template <int W, int NT, int NW, typename OT>
__global__ void __launch_bounds__(NW * 32, kSmWarps / NW)
    kv4_attention_kernel(const __grid_constant__ Kv4AttnParams p) {
    constexpr int kWarps = NW, kThreads = NW * 32;
    constexpr uint32_t kTile = NW * kTurn;  // positions of one block's turn
    constexpr uint32_t S = 4 * NT;
    constexpr uint32_t HP = 32 * W;
    constexpr uint32_t ROW = 16 * W;  // bytes of a row of codes
    constexpr uint32_t PART = S * (HP + 2);
    constexpr uint32_t M0 = 0x000f000fu, M1 = 0x00f000f0u;
    // Columns of the weights. For f32 outputs a slot has two, the whole number and the rest. For
    // bf16 outputs it has one, the weight rounded to fp16 (2^-12 of it, an eighth of the output's
    // own rounding), and two sets of four slots share one operand.
    constexpr bool F32 = sizeof(OT) == 4;
    constexpr int NA = F32 ? NT : 1;
    // Sums of bf16 outputs stay in the unit's accumulators. Those of f32 outputs start from zero
    // every turn and are added to running ones, the rest's with the whole numbers', outside: the
    // unit's own addition cuts off, and over a chain of positive terms that shows (5e-6 over 9
    // turns, 1.4e-5 over 28, 2.4e-4 over 1953, the 500000 positions of a block).
    constexpr bool KEEP = !F32;
    using St = Stage<W>;
    constexpr uint32_t RING = kStages * St::BYTES;  // a warp's turns
    constexpr uint32_t QF = NT * W * 2 * 32;        // operand words (uint2) of a unit's queries
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float s_m[kWarps][S], s_l[kWarps][S];
    __shared__ Slot s_slot[2][S];
    __shared__ Span s_span[3];
    __shared__ Job s_job[2];
    __shared__ uint32_t s_scan[kWarps], s_begin, s_end, s_item, s_at, s_jobs;

    const uint32_t tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    pdl_wait();
    pdl_trigger();
    const uint32_t r = lane / 4, c = lane % 4;
    unsigned char* ring = smem + warp * RING;
    float* so = reinterpret_cast<float*>(smem + kWarps * RING);  // outputs [kWarps][S][HP]
    // the queries' operand columns, of this unit and the next
    uint2* s_q = reinterpret_cast<uint2*>(smem + kWarps * (RING + S * HP * 4));

    // ---- this block's stretch of the line --------------------------------------------------
    if (blockIdx.x == 0) {
        for (uint32_t i = tid; i < p.rows; i += kThreads)
            if (p.step[i].position >= p.c.seq) atomicOr(p.flags, kFlagPositionRange);
    }
    uint32_t total = 0;  // tiles in all
    if (p.items == 1) {
        if (warp == 0) total = (tiles_of<NW>(item_length<S>(p, 0)) + p.lead) * p.per_item;
    } else {
        uint32_t sum = 0;
        for (uint32_t i = tid; i < p.items; i += kThreads)
            sum += tiles_of<NW>(item_length<S>(p, i)) + p.lead;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) s_scan[warp] = sum;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; w++) total += s_scan[w];
        total *= p.per_item;
    }
    // Scalar work on the line is the first warp's; the others read what it found.
    Line line;
    if (warp == 0) {
        line = Line(total, gridDim.x);
        if (lane == 0) {
            const bool any = blockIdx.x < line.blocks;
            s_begin = any ? line.begin(blockIdx.x) : total;
            s_end = any ? line.begin(blockIdx.x + 1) : total;
        }
    }
    __syncthreads();
    const uint32_t begin = s_begin, end = s_end;
    if (begin >= end) return;
    uint32_t item = 0, item_at = 0;  // tiles before `item`
    if (p.items > 1) {
        uint32_t base = 0;
        for (uint32_t i0 = 0; i0 < p.items; i0 += kThreads) {
            const uint32_t i = i0 + tid;
            const uint32_t n =
                i < p.items ? (tiles_of<NW>(item_length<S>(p, i)) + p.lead) * p.per_item : 0;
            uint32_t upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= (uint32_t)o) upto += x;
            }
            __syncthreads();
            if (lane == 31) s_scan[warp] = upto;
            __syncthreads();
            upto += base;
#pragma unroll
            for (uint32_t w = 0; w < kWarps; w++) {
                if (w < warp) upto += s_scan[w];
                base += s_scan[w];
            }
            if (begin < upto && begin >= upto - n) {
                s_item = i;
                s_at = upto - n;
            }
            if (base > begin) break;
        }
        __syncthreads();
        item = s_item;
        item_at = s_at;
    }

    // The units of the stretch overlap: while one's positions are computed, the next one's place
    // in the line is found and its queries are read; its first turns are on their way while the
    // warps' parts are joined.
    uint32_t len = 0, len1 = 0, n_tiles = 0, jobs = 0;  // len1: of the item after
    if (warp == 0) {
        len = item_length<S>(p, item);
        len1 = item + 1 < p.items ? item_length<S>(p, item + 1) : 0;
        n_tiles = tiles_of<NW>(len);
    }
    auto plan = [&](uint32_t at, Span& span) {  // the unit at `at`: the first warp's work
        while (at - item_at >= (n_tiles + p.lead) * p.per_item) {
            item_at += (n_tiles + p.lead) * p.per_item;
            item++;
            len = len1;
            len1 = item + 1 < p.items ? item_length<S>(p, item + 1) : 0;
            n_tiles = tiles_of<NW>(len);
        }
        const uint32_t nth = (at - item_at) / (n_tiles + p.lead);
        if (lane == 0) {
            span.item = item;
            span.nth = nth;
            span.sub = nth / p.c.kv_heads;
            span.kvh = nth - span.sub * p.c.kv_heads;
            span.at = item_at + nth * (n_tiles + p.lead) + p.lead;
            span.until = span.at + n_tiles;
            span.t_begin = (max(at, span.at) - span.at) * kTile;
            span.t_end = min((min(end, span.until) - min(end, span.at)) * kTile, len);
        }
    };
    const unsigned char *ksrc, *vsrc;
    const uint32_t *kscale, *vscale;
    uint32_t t, t_end, stage = 0;
    // The warp's turn at t into stage i, one group of copies (an empty one past the end).
    // Chunk lane + 32 j is chunk (lane + 32 j) % W of row (lane + 32 j) / W.
    auto fetch = [&](uint32_t t, uint32_t i) {
        const uint32_t to = smem_u32(ring) + i * St::BYTES;
        const unsigned char* k = ksrc + (uint64_t)t * ROW;
        const unsigned char* v = vsrc + (uint64_t)t * ROW;
        auto copy = [&](uint32_t n) {  // of n rows
#pragma unroll
            for (uint32_t j = 0; j < W; j++) {
                const uint32_t row = (lane + 32 * j) / W;
                const uint32_t at = to + St::place(row, (lane + 32 * j) % W);
                const uint32_t size = row < n ? 16 : 0;
                copy16(at, k + (size ? j * 512 : 0), size);
                copy16(at + St::V, v + (size ? j * 512 : 0), size);
            }
            const uint32_t size = lane < n ? 4 : 0;
            copy4(to + St::KS + 4 * lane, kscale + (size ? t : 0), size);
            copy4(to + St::VS + 4 * lane, vscale + (size ? t : 0), size);
        };
        if (t + kTurn <= t_end) copy(kTurn);
        else if (t < t_end) copy(t_end - t);
        copies_commit();
    };
    auto open = [&](const Span& span) {  // the unit's first turns
        const uint64_t vec0 = (uint64_t)(p.shared ? 0 : span.item) * p.c.row_stride +
                              (uint64_t)span.kvh * p.c.seq;
        ksrc = (const unsigned char*)p.c.codes[0] + vec0 * ROW + lane * 16;
        vsrc = (const unsigned char*)p.c.codes[1] + vec0 * ROW + lane * 16;
        kscale = p.c.scales[0] + vec0 + lane;
        vscale = p.c.scales[1] + vec0 + lane;
        t_end = span.t_end;
        t = span.t_begin + warp * kTurn;
#pragma unroll 1
        for (uint32_t i = 0; i < kStages; i++) fetch(t + i * kTile, (stage + i) % kStages);
    };
    // Queries, times log2(e) / sqrt(head), as operand columns: column 2 (s % 4) of slot s is the
    // whole number next to q 2^e, the next one the rest; e brings the head's largest |q| to
    // [2^10, 2^11). Warp w takes slots w, w + NW, .. , a lane four dims.
    constexpr uint32_t TAKES = (S + NW - 1) / NW;
    float qx[TAKES][4];
    int32_t qlimit[TAKES];
    auto read_queries = [&](const Span& span) {
#pragma unroll
        for (uint32_t j = 0; j < TAKES; j++) {
            const uint32_t s = warp + NW * j;
            if (s >= S) return;
            float(&x)[4] = qx[j];
            uint32_t row, head;
            const bool live =
                Unit<W, S, OT>{p, span.item, span.kvh, span.sub}.slot(s, &row, &head);
            const uint32_t d0 = lane * 4, hd = p.c.head;
            x[0] = x[1] = x[2] = x[3] = 0.0f;
            if (live && d0 < hd) {
                const float* src = p.q + ((uint64_t)row * p.heads + head) * hd + d0;
                if (p.qvec) {
                    const uint4 a = ld16(src);
                    x[0] = __uint_as_float(a.x); x[1] = __uint_as_float(a.y);
                    x[2] = __uint_as_float(a.z); x[3] = __uint_as_float(a.w);
                } else {
#pragma unroll
                    for (uint32_t k = 0; k < 4; k++)
                        if (d0 + k < hd) x[k] = __uint_as_float(ld4(src + k));
                }
            }
            // past the last slot: nothing of it is written
            qlimit[j] = live ? (int32_t)min(p.step[row].position, 0x7fffffffu) : 0x7fffffff;
            if (live && qlimit[j] >= (int32_t)p.c.seq) qlimit[j] = -1;
        }
    };
    auto set_queries = [&](uint2* qf, Slot* slots) {
        const float unit_scale = kLog2e / sqrtf((float)p.c.head);
#pragma unroll
        for (uint32_t j = 0; j < TAKES; j++) {
            const uint32_t s = warp + NW * j;
            if (s >= S) return;
            float(&x)[4] = qx[j];
            float top = 0.0f, sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                x[k] *= unit_scale;
                top = fmaxf(top, fabsf(x[k]));
                sum += x[k];
            }
            top = warp_max(top);
            int e = 10 - ((int)(__float_as_uint(top) >> 23) - 127);
            e = min(max(e, -100), 100);
            const float up = __uint_as_float((uint32_t)(e + 127) << 23);
            float first = 0.0f, rest = 0.0f;
            const uint32_t word = lane / 2, col = 2 * (s % 4);
            __half* dst = reinterpret_cast<__half*>(qf) + lane % 2;
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) {
                const float v = x[k] * up, w = rintf(v);  // the rest is NaN where q is not finite
                first += w;
                rest += v - w;
                if (word < 4 * W) {
                    // code k of a half word is at bits 4 k: even k as c 2^-24, odd as 16 c 2^-24
                    const uint32_t at = (((s / 4) * W + word % W) * 2 + k / 2) * 32 + word / W;
                    const float f = k % 2 ? 0.0625f : 1.0f;
                    dst[((at + col * 4) * 2 + k % 2) * 2] = __float2half_rn(w * f);
                    dst[((at + col * 4 + 4) * 2 + k % 2) * 2] = __float2half_rn((v - w) * f);
                }
            }
            sum = warp_sum(sum);
            first = warp_sum(first);
            rest = warp_sum(rest);
            if (lane == 0)
                slots[s] = Slot{16777216.0f / up, sum, first * (-8.0f / 16777216.0f),
                                rest * (-8.0f / 16777216.0f), qlimit[j]};
        }
    };

    if (warp == 0) plan(begin, s_span[0]);
    __syncthreads();
    if (s_span[0].at >= end) return;  // of its lead alone
    open(s_span[0]);
    read_queries(s_span[0]);
    set_queries(s_q, s_slot[0]);
    for (uint32_t nth = 0;; nth++) {
        const Span& span = s_span[nth % 3];
        Span& after = s_span[(nth + 1) % 3];
        const uint32_t next_at = min(end, span.until);
        const bool more = next_at + p.lead < end;
        if (more && warp == 0) plan(next_at, after);
        __syncthreads();  // this unit's queries, the next one's place; the last one's outputs are read
        if (more) read_queries(after);
        const uint2* qf = s_q + nth % 2 * QF;
        float qscale[NT], qsum[NT], qmid[NT][2];  // of slot c (+ 4 nt)
        int32_t limit[NT], lowest = 0x7fffffff;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const Slot& q = s_slot[nth % 2][c + 4 * nt];
            qscale[nt] = q.scale;
            qsum[nt] = q.sum;
            qmid[nt][0] = q.first;
            qmid[nt][1] = q.rest;
            limit[nt] = q.limit;
            lowest = min(lowest, q.limit);
        }
        lowest = min(lowest, __shfl_xor_sync(0xffffffffu, lowest, 1));
        lowest = min(lowest, __shfl_xor_sync(0xffffffffu, lowest, 2));

        // ---- the positions -----------------------------------------------------------------
        // Weights are w = 2^(score - M). M is the largest score + log2 g so far, less TOP, moved when
        // a w x g reaches 2^11; g is the step of V where that is not small. As for the queries, the
        // whole number of w x step is one operand column, exact in the sums, and the rest, 11 bits
        // of at most a half, the other. With TOP 9 f32 outputs of 100 positions were up to 1.1e-6
        // off, with 10 some 6e-7 on the same inputs. g is at least a 2^-20th of the offset, so that
        // 2^31 terms w x offset are below 2^63 (a step below that adds less than the offset's own
        // rounding), and at least kLeast, so that as many weights are below 2^126. (A bound on
        // w x step alone let the weights of vectors without a step overflow; this one costs 1 to 2%
        // at many short units, 43.3 to 44.2 us at 256 streams, nothing at one long row.)
        constexpr float kLeast = 0x1p-84f;
        constexpr float TOP = F32 ? 10.0f : 9.0f;
        float o[NT][2 * W][2], kept[NA][2 * W][4], l[NT], pm[NT], M[NT], cap[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            l[nt] = pm[nt] = M[nt] = 0.0f;
            cap[nt] = -1.0f;  // no position yet: any moves M
#pragma unroll
            for (int i = 0; i < 2 * W; i++) o[nt][i][0] = o[nt][i][1] = 0.0f;
        }
#pragma unroll
        for (int n = 0; n < NA; n++)
#pragma unroll
            for (int i = 0; i < 2 * W; i++)
                kept[n][i][0] = kept[n][i][1] = kept[n][i][2] = kept[n][i][3] = 0.0f;
        // Position 8 i + r of the 32, i = 0 .. 3, is lane r's: row r (even i) or 8 + r of the
        // operand of K's mma i / 2; V's takes the rows in the same order.
        const uint32_t k_at = W == 4   ? St::place(r, c)
                              : W == 2 ? St::place(r, c / 2) + c % 2 * 8
                                       : r * ROW + c * 4 * W;
        for (; t < t_end; t += kTile) {
            copies_wait<kStages - 1>();
            __syncwarp();
            const uint32_t st = smem_u32(ring) + stage * St::BYTES;
            uint32_t ks[4], vs[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                ks[i] = lds4(st + St::KS + 4 * r + 32 * i);
                vs[i] = lds4(st + St::VS + 4 * r + 32 * i);
            }
            float acc[2][NT][4];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                uint32_t kw[2][W];
#pragma unroll
                for (int h = 0; h < 2; h++) load_k<W>(st + k_at + (16 * i + 8 * h) * ROW, kw[h]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    acc[i][nt][0] = acc[i][nt][2] = qmid[nt][0];
                    acc[i][nt][1] = acc[i][nt][3] = qmid[nt][1];
                }
#pragma unroll
                for (int w = 0; w < W; w++) {
                    const uint32_t x0 = kw[0][w], x1 = kw[1][w];
                    const uint32_t y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        const uint2 b0 = qf[(nt * W + w) * 64 + lane],
                                    b1 = qf[(nt * W + w) * 64 + 32 + lane];
                        mma16816(acc[i][nt], x0 & M0, x1 & M0, x0 & M1, x1 & M1, b0.x, b0.y);
                        mma16816(acc[i][nt], y0 & M0, y1 & M0, y0 & M1, y1 & M1, b1.x, b1.y);
                    }
                }
            }
            float g[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                g[i] = fmaxf(fmaxf(bf16lo(vs[i]), fabsf(bf16hi(vs[i])) * 0x1p-20f), kLeast);
            // score - M = s (q . (c - 8)) + (m + 8 s) sum q - M, taken off M first: the exact
            // whole-number sum meets it inside one rounding, at the size of the difference, so a
            // large score costs the weights no digits
            float sc[NT][4], w[NT][4], ws[NT][4];
            bool over = false;
            auto weigh = [&](auto masked) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float step = bf16lo(ks[i]), sq = step * qscale[nt];
                        float x = fmaf(acc[i / 2][nt][2 * (i % 2)], sq, -M[nt]);
                        x = fmaf(fmaf(8.0f, step, bf16hi(ks[i])), qsum[nt], x);
                        x = fmaf(acc[i / 2][nt][2 * (i % 2) + 1], sq, x);
                        const bool out = masked.value && (int32_t)(t + 8 * i + r) > limit[nt];
                        sc[nt][i] = out ? -INFINITY : x;
                        w[nt][i] = ex2(sc[nt][i]);
                        ws[nt][i] = out ? 0.0f : w[nt][i] * bf16lo(vs[i]);
                    }
                    over |= fmaxf(fmaxf(w[nt][0] * g[0], w[nt][1] * g[1]),
                                  fmaxf(w[nt][2] * g[2], w[nt][3] * g[3])) > cap[nt];
                }
            };
            const bool masked = (int32_t)(t + kTurn - 1) > lowest;
            if (masked) weigh(std::true_type());
            else weigh(std::false_type());
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float top = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int e = (int)(__float_as_uint(g[i]) >> 23) - 127;
                        top = fmaxf(top, sc[nt][i] + (float)e);
                    }
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1)
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    if (top > (cap[nt] < 0.0f ? -INFINITY : TOP)) {
                        const float to = M[nt] + (top - TOP), a = ex2(M[nt] - to);
                        M[nt] = to;
                        if (cap[nt] > 0.0f) {
                            l[nt] *= a;
                            pm[nt] *= a;
#pragma unroll
                            for (int i = 0; i < 2 * W; i++) {
                                if constexpr (F32) {
                                    o[nt][i][0] *= a;
                                    o[nt][i][1] *= a;
                                } else {
                                    kept[0][i][nt] *= a;
                                    kept[0][i][2 + nt] *= a;
                                }
                            }
                        }
                        cap[nt] = 2048.0f;
                    }
                }
                weigh(std::true_type());
            }
            uint32_t pb[NA][4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    l[nt] += w[nt][i];
                    if (!masked || (int32_t)(t + 8 * i + r) <= limit[nt])
                        pm[nt] = fmaf(w[nt][i], bf16hi(vs[i]), pm[nt]);
                    if constexpr (F32) {
                        // the nearest whole number, by way of 1.5 2^23
                        const float first = (ws[nt][i] + 12582912.0f) - 12582912.0f;
                        const __half2 two = __floats2half2_rn(first, ws[nt][i] - first);
                        pb[nt][i] = transpose8(*reinterpret_cast<const uint32_t*>(&two));
                    }
                }
                if constexpr (!F32) {
                    const __half2 two = __floats2half2_rn(ws[0][i], NT == 2 ? ws[NT - 1][i] : 0.0f);
                    pb[0][i] = transpose8(*reinterpret_cast<const uint32_t*>(&two));
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < W; k++) {
                uint32_t y[4];
                load_v(st + St::V + St::place(lane, k), y);
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    if (b) {
#pragma unroll
                        for (int i = 0; i < 4; i++) y[i] >>= 8;
                    }
#pragma unroll
                    for (int n = 0; n < NA; n++) {
                        if constexpr (KEEP) {
                            float (&a)[4] = kept[n][2 * k + b];
                            mma16816(a, y[0] & M0, y[0] & M1, y[1] & M0, y[1] & M1, pb[n][0],
                                     pb[n][1]);
                            mma16816(a, y[2] & M0, y[2] & M1, y[3] & M0, y[3] & M1, pb[n][2],
                                     pb[n][3]);
                        } else {
                            float a[4];
                            mma16816_zero(a, y[0] & M0, y[0] & M1, y[1] & M0, y[1] & M1, pb[n][0],
                                          pb[n][1]);
                            mma16816(a, y[2] & M0, y[2] & M1, y[3] & M0, y[3] & M1, pb[n][2],
                                     pb[n][3]);
                            o[n][2 * k + b][0] += a[0] + a[1];
                            o[n][2 * k + b][1] += a[2] + a[3];
                        }
                    }
                }
            }
            __syncwarp();  // every lane is done with the stage
            fetch(t + kStages * kTile, stage);
            stage = (stage + 1) % kStages;
        }

        if constexpr (KEEP) {
            // rows r and 8 + r of columns 2 c (slot c) and 2 c + 1 (slot c + 4)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 2 * W; i++) {
                    o[nt][i][0] = kept[0][i][nt];
                    o[nt][i][1] = kept[0][i][2 + nt];
                }
        }
        if (more) {
            open(after);
            set_queries(s_q + (nth + 1) % 2 * QF, s_slot[(nth + 1) % 2]);
        }

        // ---- the warps' parts joined -----------------------------------------------------------
        float* mo = so + warp * (S * HP);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) {
                l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], s);
                pm[nt] += __shfl_xor_sync(0xffffffffu, pm[nt], s);
            }
            if (r == 0) {
                // no positions: no part (a sum that is NaN is one)
                s_m[warp][c + 4 * nt] = l[nt] == 0.0f ? -INFINITY : M[nt];
                s_l[warp][c + 4 * nt] = l[nt];
            }
#pragma unroll
            for (int i = 0; i < 2 * W; i++) {
                const uint32_t d = (8 * (i / 2) + r) * 4 + 2 * (i % 2);
                *reinterpret_cast<float2*>(mo + (c + 4 * nt) * HP + d) =
                    make_float2(fmaf(o[nt][i][0], 16777216.0f, pm[nt]),
                                fmaf(o[nt][i][1], 1048576.0f, pm[nt]));
            }
        }
        __syncthreads();
        const Unit<W, S, OT> unit{p, span.item, span.kvh, span.sub};
        const bool whole = begin <= span.at && span.until <= end;
        // a unit that began in an earlier stretch is this block's first part, else its last
        float* mine = p.part + (uint64_t)(2 * blockIdx.x + (begin <= span.at)) * PART;
        for (uint32_t i = tid; i < S * HP / 4; i += kThreads) {
            const uint32_t s = i * 4 / HP, d = i * 4 % HP;
            float J = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) J = fmaxf(J, s_m[w][s]);
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float4 v = *reinterpret_cast<const float4*>(so + (w * S + s) * HP + d);
                const float a = s_m[w][s] == -INFINITY ? 0.0f : ex2(s_m[w][s] - J);
                L = fmaf(s_l[w][s], a, L);
                x.x = fmaf(v.x, a, x.x);
                x.y = fmaf(v.y, a, x.y);
                x.z = fmaf(v.z, a, x.z);
                x.w = fmaf(v.w, a, x.w);
            }
            if (whole) {
                unit.write(i, x, L);
            } else {
                __stcg(reinterpret_cast<float4*>(mine) + i, x);
                if (d == 0) {
                    __stcg(mine + S * HP + s, J);
                    __stcg(mine + S * HP + S + s, L);
                }
            }
        }
        if (!whole) {
            __syncthreads();  // the block's part is written; its first thread publishes it
            if (tid == 0) {
                // blocks first .. last meet this unit; the last to arrive joins their parts, after
                // its stretch: up to two units, those at the stretch's ends
                const uint32_t first = line.block_of(span.at);
                const uint32_t parts = line.block_of(span.until - 1) - first + 1;
                uint32_t* ticket = p.tickets + (uint64_t)unit.item * p.per_item + span.nth;
                if (kv4_arrive(ticket) == parts - 1) {
                    *ticket = 0;
                    s_job[jobs++] = Job{unit.item, unit.kvh, unit.sub, first, parts};
                }
            }
        }
        if (!more) break;
    }
    if (tid == 0) s_jobs = jobs;
    __syncthreads();
    for (uint32_t k = 0; k < s_jobs; k++) {
        const Job& job = s_job[k];
        join_parts<W, NW>(Unit<W, S, OT>{p, job.item, job.kvh, job.sub}, job.first, job.parts,
                         tid, so, s_m, s_l);
        __syncthreads();
    }
}

template <int W, int NT, int NW, typename OT>
void record_one(ab_scheme* s, const char* label, Kv4AttnParams p) {
    constexpr uint32_t S = 4 * NT, PART = S * (32 * W + 2), TILE = NW * kTurn;
    constexpr size_t smem = NW * (kStages * Stage<W>::BYTES + S * 32 * W * 4) +
                            2 * NT * W * 2 * 32 * sizeof(uint2);
    auto* kernel = kv4_attention_kernel<W, NT, NW, OT>;
    const uint64_t units = (uint64_t)p.items * p.per_item;
    const uint64_t tiles = units * ((p.c.seq + TILE - 1) / TILE);
    if ((tiles + kLead<NW> * units) >> 31) invalid("kv4_attention: too much work for one call");
    s->rt->activate();
    cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
               "kv4_attention shared memory");
    const uint32_t grid =
        (uint32_t)std::min<uint64_t>((uint64_t)s->rt->sm_count * (kSmWarps / NW), tiles);
    // with fewer units than blocks a stretch holds one or two: no difference, or 1 us lost
    p.lead = units > grid ? kLead<NW> : 0;
    kv4_take_scratch(s, (uint64_t)grid * 2 * PART * 4, units, &p.part, &p.tickets);
    s->add(label, [=](cudaStream_t stream) {
        return launch(stream, dim3(grid), dim3(NW * 32), smem, true, kernel, p);
    });
}

template <int W>
void record_width(ab_scheme* s, const char* label, Kv4AttnParams p, int32_t out_dtype) {
    // four query slots a unit where a kv head has no more, else eight
    p.shared = p.c.row_stride == 0 && p.rows > 1;
    const uint64_t slots = p.shared ? (uint64_t)p.rows * p.group : p.group;
    const uint32_t S = slots <= 4 ? 4 : 8;
    const uint32_t blocks = (uint32_t)((slots + S - 1) / S);
    p.items = p.shared ? blocks : p.rows;
    p.per_item = p.c.kv_heads * (p.shared ? 1 : blocks);
    const bool many = (uint64_t)p.items * p.per_item > (uint64_t)s->rt->sm_count * (kSmWarps / 4);
    auto record = [&](auto nt, auto nw) {
        constexpr int NT = decltype(nt)::value, NW = decltype(nw)::value;
        if (out_dtype == AB_F32) record_one<W, NT, NW, float>(s, label, p);
        else record_one<W, NT, NW, bf16>(s, label, p);
    };
    constexpr std::integral_constant<int, 1> one;
    constexpr std::integral_constant<int, 2> two;
    constexpr std::integral_constant<int, 4> four;
    constexpr std::integral_constant<int, 8> eight;
    if (S == 4) {
        many ? record(one, four) : record(one, eight);
    } else if constexpr (W < 4) {
        many ? record(two, four) : record(two, eight);
    } else {
        record(two, eight);
    }
}

}  // namespace

void kv4_take_scratch(ab_scheme* s, uint64_t part_bytes, uint64_t tickets, float** part,
                      uint32_t** ticket) {
    auto& have = s->kv4;
    if (have.part_bytes < part_bytes) {
        void* d = nullptr;
        cuda_check(cudaMalloc(&d, part_bytes), "cudaMalloc");
        s->owned.push_back(d);
        have.part = d;
        have.part_bytes = part_bytes;
    }
    if (have.tickets_n < tickets) {
        void* d = nullptr;
        cuda_check(cudaMalloc(&d, tickets * 4), "cudaMalloc");
        s->owned.push_back(d);
        cuda_check(clear_device(s->rt, d, tickets * 4), "clear tickets");
        have.tickets = (uint32_t*)d;
        have.tickets_n = tickets;
    }
    *part = (float*)have.part;
    *ticket = have.tickets;
}

void record_kv4_attention(ab_scheme* s, const char* label, const float* q, uint32_t rows,
                          uint32_t heads, const Kv4View& cache, void* out, int32_t out_dtype,
                          const Step* step) {
    const uint32_t head = cache.head;
    if ((uint64_t)rows * heads > 1u << 30) invalid("parameter `q`: too many rows");
    if (cache.seq > 0x7fffff00u) invalid("parameter `cache.key_codes`: seq exceeds 2^31 - 256");
    if ((uintptr_t)q % 4 || (uintptr_t)out % dtype_size(out_dtype))
        invalid("parameter `q` / `out`: not aligned to its elements");
    if (!s->rt)
        fail(AB_ERR_ARGUMENT, "kv4_attention: the scheme needs a runtime (it allocates the split "
                              "scratch)");
    const uint64_t slots = (uint64_t)rows * (heads / cache.kv_heads);  // over one shared cache
    if (cache.row_stride == 0 && out_dtype == AB_BF16 && slots > kTensorSlots &&
        record_kv4_prompt_tc(s, label, q, rows, heads, cache, out, step))
        return;
    Kv4AttnParams p = {};
    p.c = cache;
    p.q = q;
    p.out = out;
    p.rows = rows;
    p.heads = heads;
    p.group = heads / cache.kv_heads;
    p.qvec = head % 4 == 0 && (uintptr_t)q % 16 == 0;
    p.ovec = head % 4 == 0 && (uintptr_t)out % (4 * dtype_size(out_dtype)) == 0;
    p.step = step;
    p.flags = s->rt->flags;
    switch (cache.words / 4) {
        case 1: record_width<1>(s, label, p, out_dtype); break;
        case 2: record_width<2>(s, label, p, out_dtype); break;
        case 3: record_width<3>(s, label, p, out_dtype); break;
        default: record_width<4>(s, label, p, out_dtype); break;
    }
}

}  // namespace ab

using namespace ab;

extern "C" int ab_kernel_kv4_attention(ab_scheme* s, ab_tensor q, const ab_kv4_layer* cache,
                                       ab_tensor out, ab_tensor step) {
    return guard([&] {
        if (!s || !cache) fail(AB_ERR_ARGUMENT, "null argument");
        expect_data("q", q);
        expect_data("out", out);
        expect_dtype("q", q, AB_F32);
        expect_rank_in("q", q, 2, 3);
        expect_float("out", out);
        const uint32_t rows = q.rank == 3 ? q.dims[0] : 1;
        const uint32_t heads = q.dims[q.rank - 2], head = q.dims[q.rank - 1];
        expect_data("cache.key_codes", cache->key_codes);
        expect_rank_in("cache.key_codes", cache->key_codes, 3, 4);
        const uint32_t kv = cache->key_codes.dims[cache->key_codes.rank - 3];
        if (heads % kv)
            invalid("parameter `cache.key_codes`: kv_heads " + std::to_string(kv) +
                    " must divide the " + std::to_string(heads) + " query heads");
        const Kv4View c = kv4_operands(*cache, rows, kv, head);
        if (numel(out) != (uint64_t)rows * heads * head)
            invalid("parameter `out`: expected " +
                    std::to_string((uint64_t)rows * heads * head) +
                    " elements ([batch, heads * head]), got " + shape_str(out));
        expect_step(step, rows);
        const uintptr_t q0 = (uintptr_t)q.data, o0 = (uintptr_t)out.data;
        if (q0 < o0 + numel(out) * dtype_size(out.dtype) && o0 < q0 + numel(q) * 4)
            invalid("parameter `out`: overlaps q");
        record_kv4_attention(s, "kv4_attention", (const float*)q.data, rows, heads, c, out.data,
                             out.dtype, (const Step*)step.data);
    });
}
