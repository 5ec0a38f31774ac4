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
// is the 16-row operand (16 positions for K, 16 dims for V), read once for all query heads of
// its group; the queries and the weights are the 8-column one, each head taking two columns of
// fp16, the whole number and the rest, together 22 bits. So f32 results keep their digits, and one
// lane's accumulators all belong to one head: its maximum, sum and rescaling need no exchange.
//
// Bound: the packed bytes. A warp's 32 positions (head 128) are 4352 bytes and about 400
// instructions; a twelfth of them is mma. K, V and scales of the next 32 positions load into
// registers straight from global memory while the present ones are computed.
//
// Split: the tiles of all units (a row's or a slot block's positions of one kv head) form one
// line that the teams of one wave of blocks share equally, so rows of unlike lengths and few
// rows of great length fill the device alike. A team is a block's eight warps, 32 positions
// each at a time, where units are few and long; a warp where they are many, so that short rows
// do not pay for eight warps' start and joining. A unit that several teams meet is joined by
// the last of them to finish, in line order: results do not depend on which that is.
#include <cuda_fp16.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "kv4.h"

namespace ab {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr uint32_t kTurn = 32;   // positions of one warp's turn
constexpr float kLog2e = 1.4426950408889634f;

struct Kv4AttnParams {
    const float* q;  // [rows, heads, head]
    void* out;       // [rows, heads * head]
    Kv4View c;
    uint32_t rows, heads, group;
    uint32_t items;     // rows with a cache each, or blocks of query slots over one cache
    uint32_t per_item;  // kv heads x slot blocks of a row's group
    int shared;         // rows share one cache
    int qvec, svec, ovec;  // 16-byte loads of q and of four scale words, four outputs at once
    float* part;        // [2 teams][slots][32 W + 2] partial results
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
__device__ __forceinline__ uint2 ld8(const void* p) {
    uint2 r;
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];"
                 : "=r"(r.x), "=r"(r.y)
                 : "l"(p));
    return r;
}
__device__ __forceinline__ uint32_t ld4(const void* p) {
    uint32_t r;
    asm volatile("ld.global.u32 %0, [%1];" : "=r"(r) : "l"(p));
    return r;
}
__device__ __forceinline__ uint32_t ld2(const void* p) {
    uint16_t r;
    asm volatile("ld.global.u16 %0, [%1];" : "=h"(r) : "l"(p));
    return r;
}

// W words: a lane's quarter of a K row.
template <int W>
__device__ __forceinline__ void load_k(const unsigned char* p, uint32_t (&w)[W]) {
    if constexpr (W == 4) {
        const uint4 r = ld16(p);
        w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
    } else if constexpr (W == 2) {
        const uint2 r = ld8(p);
        w[0] = r.x; w[1] = r.y;
    } else {
#pragma unroll
        for (int i = 0; i < W; i++) w[i] = ld4(p + 4 * i);
    }
}

// A lane's eighth of a V row: W units of 16 bits (four dims each), two to a word where the
// address allows (even W), else one.
template <int W>
constexpr int kVWords = W % 2 == 0 ? W / 2 : W;
template <int W>
__device__ __forceinline__ void load_v(const unsigned char* p, uint32_t (&w)[kVWords<W>]) {
    if constexpr (W == 4) {
        const uint2 r = ld8(p);
        w[0] = r.x; w[1] = r.y;
    } else if constexpr (W == 2) {
        w[0] = ld4(p);
    } else {
#pragma unroll
        for (int i = 0; i < W; i++) w[i] = ld2(p + 2 * i);
    }
}
// Unit k of two rows side by side.
template <int W>
__device__ __forceinline__ uint32_t pair_units(const uint32_t (&a)[kVWords<W>],
                                               const uint32_t (&b)[kVWords<W>], int k) {
    if constexpr (W % 2 == 0)
        return __byte_perm(a[k / 2], b[k / 2], k % 2 ? 0x7632 : 0x5410);
    else
        return __byte_perm(a[k], b[k], 0x5410);
}

// One arrival at a ticket: what the block wrote before its last barrier is published with it,
// what the earlier arrivals published is seen after it.
__device__ __forceinline__ uint32_t arrive(uint32_t* ticket) {
    uint32_t before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                 : "=r"(before)
                 : "l"(ticket)
                 : "memory");
    return before;
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
// Tiles of TILE positions; at least one, so that a row without positions is written too.
template <uint32_t TILE>
__device__ __forceinline__ uint32_t tiles_of(uint32_t length) {
    return max(1u, (length + TILE - 1) / TILE);
}

// The line of `total` tiles over `teams` teams: the first `more` of them take one tile more.
struct Line {
    uint32_t teams = 0, each = 0, more = 0;
    __device__ __forceinline__ Line() {}
    __device__ __forceinline__ Line(uint32_t total, uint32_t most) {
        teams = min(total, most);
        each = total / teams;
        more = total % teams;
    }
    __device__ __forceinline__ uint32_t begin(uint32_t team) const {
        return team * each + min(team, more);
    }
    __device__ __forceinline__ uint32_t team_of(uint32_t tile) const {
        const uint32_t cut = more * (each + 1);
        return tile < cut ? tile / (each + 1) : more + (tile - cut) / each;
    }
};

// What a team's first warp finds for all: its stretch, the unit at hand (tiles [at, until) of
// the line) and the part of it that is the team's.
struct Span {
    uint32_t begin, end;
    uint32_t item, nth, kvh, sub, at, until, t_begin, t_end;
};

// A unit whose parts, those of teams first .. first + parts - 1, are to be joined.
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

template <int TEAM>
__device__ __forceinline__ void team_sync() {
    if constexpr (TEAM == 1) __syncwarp();
    else __syncthreads();
}

// Joins the parts of teams first .. first + n - 1 in that order and writes the unit's rows.
// [S][32 W] outputs are COLS groups of four; where these are fewer than the team's TT threads,
// JG threads share one and take every JG-th part (what is left of the threads rests). A thread
// joins its parts as an online softmax does, so that weights and values are read in one round,
// AHEAD parts at a time. so, sm, sl: the team's shared arrays, free by now.
template <int W, uint32_t S, int TEAM, typename OT>
__device__ __forceinline__ void join_parts(const Unit<W, S, OT>& unit, uint32_t first, uint32_t n,
                                        uint32_t tt, float4* so, float (*sm)[S], float (*sl)[S]) {
    constexpr uint32_t PART = S * (32 * W + 2), COLS = S * 8 * W, TT = TEAM * 32;
    constexpr uint32_t JG = COLS < TT ? TT / COLS : 1;
    constexpr uint32_t PER = COLS < TT ? 1 : COLS / TT;
    constexpr uint32_t AHEAD = PER == 1 ? 8 : PER <= 4 ? 3 : 2;
    static_assert(JG <= TEAM, "what a column's threads exchange fits where the warps' parts were");
    const uint32_t col = tt % COLS, jg = COLS < TT ? tt / COLS : 0;
    float4 x[PER];
    float J[PER], L[PER];
#pragma unroll
    for (uint32_t k = 0; k < PER; k++) {
        x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        J[k] = -INFINITY;
        L[k] = 0.0f;
    }
    auto join = [&](uint32_t k, const float4& v, float mj, float lj) {
        if (mj == -INFINITY) return;
        const float to = fmaxf(J[k], mj), a = ex2(J[k] - to), b = ex2(mj - to);
        x[k].x = fmaf(v.x, b, x[k].x * a);
        x[k].y = fmaf(v.y, b, x[k].y * a);
        x[k].z = fmaf(v.z, b, x[k].z * a);
        x[k].w = fmaf(v.w, b, x[k].w * a);
        L[k] = fmaf(lj, b, L[k] * a);
        J[k] = to;
    };
    for (uint32_t j0 = jg < JG ? jg : n; j0 < n; j0 += AHEAD * JG) {
        float4 v[AHEAD][PER];
        float mj[AHEAD][PER], lj[AHEAD][PER];
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; u++) {
            const uint32_t j = j0 + u * JG;
            // the unit begins inside the first team's stretch and before the others'
            const float* pj = unit.p.part + ((uint64_t)2 * (first + j) + (j == 0)) * PART;
#pragma unroll
            for (uint32_t k = 0; k < PER; k++) {
                const uint32_t i = col + k * TT, s = i / (8 * W);
                mj[u][k] = -INFINITY;
                if (j < n) {
                    mj[u][k] = __ldcg(pj + COLS * 4 + s);
                    lj[u][k] = __ldcg(pj + COLS * 4 + S + s);
                    v[u][k] = __ldcg(reinterpret_cast<const float4*>(pj) + i);
                }
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; u++)
#pragma unroll
            for (uint32_t k = 0; k < PER; k++) join(k, v[u][k], mj[u][k], lj[u][k]);
    }
    if constexpr (JG > 1) {
        if (jg < JG) {
            so[jg * COLS + col] = x[0];
            sm[jg][col / (8 * W)] = J[0];  // the same from every thread of a slot
            sl[jg][col / (8 * W)] = L[0];
        }
        team_sync<TEAM>();
        if (jg == 0) {
#pragma unroll
            for (uint32_t g = 1; g < JG; g++)
                join(0, so[g * COLS + col], sm[g][col / (8 * W)], sl[g][col / (8 * W)]);
        }
    }
    if (jg == 0) {
#pragma unroll
        for (uint32_t k = 0; k < PER; k++) unit.write(col + k * TT, x[k], L[k]);
    }
}

// W: words of codes in a quarter row (head up to 32 W). NT: four query slots each. TEAM: warps
// that take a stretch of the line together (1 or 8).
template <int W, int NT, int TEAM, typename OT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1)
    kv4_attention_kernel(const __grid_constant__ Kv4AttnParams p) {
    constexpr uint32_t S = 4 * NT;
    constexpr uint32_t HP = 32 * W;
    constexpr uint32_t ROW = 16 * W;  // bytes of a row of codes
    constexpr uint32_t PART = S * (HP + 2);
    constexpr uint32_t TILE = TEAM * kTurn;
    constexpr uint32_t TEAMS = kWarps / TEAM, TT = TEAM * 32;  // teams of a block, their threads
    constexpr uint32_t M0 = 0x000f000fu, M1 = 0x00f000f0u;
    __shared__ float s_o[kWarps][S][HP];
    __shared__ float s_m[kWarps][S], s_l[kWarps][S];
    __shared__ float s_jm[TEAMS][S], s_jl[TEAMS][S];
    __shared__ uint2 s_q[TEAM == 1 ? 1 : NT * W * 2][32];
    __shared__ Slot s_slot[TEAMS][S];
    __shared__ Span s_span[TEAMS];
    __shared__ uint32_t s_scan[kWarps], s_item[TEAMS], s_at[TEAMS], s_jobs[TEAMS];
    __shared__ Job s_job[TEAMS][2];

    pdl_wait();
    pdl_trigger();
    const uint32_t tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const uint32_t mate = warp % TEAM, crew = warp / TEAM, tt = tid % TT;
    const uint32_t r = lane / 4, c = lane % 4;
    float (*so)[S][HP] = s_o + crew * TEAM;
    float (*sm)[S] = s_m + crew * TEAM;
    float (*sl)[S] = s_l + crew * TEAM;
    Slot* slots = s_slot[crew];
    Span& span = s_span[crew];
    // the queries' operand columns; a lone warp keeps them where its outputs go later
    uint2 (*qf)[32] = s_q;
    if constexpr (TEAM == 1) {
        static_assert(NT * W * 2 * 32 * sizeof(uint2) <= S * HP * sizeof(float), "q fits");
        qf = reinterpret_cast<uint2 (*)[32]>(&so[0][0][0]);
    }

    // ---- this team's stretch of the line --------------------------------------------------
    if (blockIdx.x == 0) {
        for (uint32_t i = tid; i < p.rows; i += kThreads)
            if (p.step[i].position >= p.c.seq) atomicOr(p.flags, kFlagPositionRange);
    }
    uint32_t total = 0;  // tiles in all
    if (p.items == 1) {
        if (mate == 0) total = tiles_of<TILE>(item_length<S>(p, 0)) * p.per_item;
    } else {
        uint32_t sum = 0;
        for (uint32_t i = tid; i < p.items; i += kThreads)
            sum += tiles_of<TILE>(item_length<S>(p, i));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) s_scan[warp] = sum;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; w++) total += s_scan[w];
        total *= p.per_item;
    }
    // Scalar work on the line is the team's first warp's; the others read what it found.
    Line line;
    const uint32_t team = blockIdx.x * TEAMS + crew;
    if (mate == 0) {
        line = Line(total, gridDim.x * TEAMS);
        if (lane == 0) {
            span.begin = team < line.teams ? line.begin(team) : total;
            span.end = team < line.teams ? line.begin(team + 1) : total;
        }
    }
    if (TEAM > 1 || p.items > 1) __syncthreads();
    else __syncwarp();
    const uint32_t begin = span.begin, end = span.end;
    uint32_t item = 0, item_at = 0;  // tiles before `item`
    if (p.items > 1) {
        uint32_t base = 0;
        for (uint32_t i0 = 0; i0 < p.items; i0 += kThreads) {
            const uint32_t i = i0 + tid;
            const uint32_t n = i < p.items ? tiles_of<TILE>(item_length<S>(p, i)) * p.per_item : 0;
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
#pragma unroll
            for (uint32_t k = 0; k < TEAMS; k++) {
                const uint32_t b = s_span[k].begin;
                if (b < upto && b >= upto - n) {
                    s_item[k] = i;
                    s_at[k] = upto - n;
                }
            }
            if (base > s_span[TEAMS - 1].begin) break;
        }
        __syncthreads();
        item = s_item[crew];
        item_at = s_at[crew];
    }

    // every later wait is a team's own
    uint32_t len = 0, n_tiles = 0, jobs = 0;
    if (begin < end && mate == 0) {
        len = item_length<S>(p, item);
        n_tiles = tiles_of<TILE>(len);
    }
    for (uint32_t at = begin; at < end;) {
        // ---- the unit (item, kv head, slot block) at `at` ---------------------------------
        if (mate == 0) {
            while (at - item_at >= n_tiles * p.per_item) {
                item_at += n_tiles * p.per_item;
                item++;
                len = item_length<S>(p, item);
                n_tiles = tiles_of<TILE>(len);
            }
            const uint32_t nth = (at - item_at) / n_tiles;
            if (lane == 0) {
                span.item = item;
                span.nth = nth;
                span.sub = nth / p.c.kv_heads;
                span.kvh = nth - span.sub * p.c.kv_heads;
                span.at = item_at + nth * n_tiles;
                span.until = span.at + n_tiles;
                span.t_begin = (at - span.at) * TILE;
                span.t_end = min((min(end, span.until) - span.at) * TILE, len);
            }
        }
        team_sync<TEAM>();
        const Unit<W, S, OT> unit{p, span.item, span.kvh, span.sub};
        const uint32_t t_end = span.t_end;
        const uint64_t vec0 = (uint64_t)(p.shared ? 0 : unit.item) * p.c.row_stride +
                              (uint64_t)unit.kvh * p.c.seq;

        // Position of index i of the 32, as an operand row: 4 r + 2 i + h of mma i, half h, for
        // K rows, scales and scores; 4 (2 c + x) + 2 i + h for V. A lane's scales are one
        // 16-byte word group.
        const unsigned char* kbase = (const unsigned char*)p.c.codes[0] + vec0 * ROW + c * (4 * W);
        const unsigned char* vbase = (const unsigned char*)p.c.codes[1] + vec0 * ROW + r * (2 * W);
        const uint32_t* ksbase = p.c.scales[0] + vec0 + 4 * r;
        const uint32_t* vsbase = p.c.scales[1] + vec0 + 4 * r;
        uint32_t kw[2][2][W], vw[2][2][2][kVWords<W>], ks[4], vs[4];
        auto load_scales = [&](const uint32_t* base, uint32_t t, uint32_t (&s)[4]) {
            if (t + kTurn <= t_end && p.svec) {
                const uint4 a = ld16(base + t);
                s[0] = a.x; s[1] = a.y; s[2] = a.z; s[3] = a.w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) s[i] = t + 4 * r + i < t_end ? ld4(base + t + i) : 0;
            }
        };
        auto load_keys = [&](uint32_t t) {
            if (t + kTurn <= t_end) {
                const unsigned char* b = kbase + (uint64_t)(t + 4 * r) * ROW;
#pragma unroll
                for (int i = 0; i < 4; i++) load_k<W>(b + i * ROW, kw[i / 2][i % 2]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    load_k<W>(kbase + (uint64_t)min(t + 4 * r + i, t_end - 1) * ROW,
                              kw[i / 2][i % 2]);
            }
            load_scales(ksbase, t, ks);
        };
        auto load_values = [&](uint32_t t) {
            if (t + kTurn <= t_end) {
                const unsigned char* b = vbase + (uint64_t)(t + 8 * c) * ROW;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    load_v<W>(b + j * ROW, vw[j / 2 % 2][j % 2][j / 4]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    load_v<W>(vbase + (uint64_t)min(t + 8 * c + j, t_end - 1) * ROW,
                              vw[j / 2 % 2][j % 2][j / 4]);
            }
            load_scales(vsbase, t, vs);
        };
        uint32_t t = span.t_begin + mate * kTurn;
        if (t < t_end) {
            load_keys(t);
            load_values(t);
        }

        // ---- queries, times log2(e) / sqrt(head), as operand columns -----------------------
        // Column 2 (s % 4) of slot s is the whole number next to q 2^e, the next one the rest;
        // e brings the head's largest |q| to [2^10, 2^11). A lane takes four dims.
        for (uint32_t s = mate; s < S; s += TEAM) {
            uint32_t row, head;
            const bool live = unit.slot(s, &row, &head);
            const uint32_t d0 = lane * 4, hd = p.c.head;
            float x[4] = {};
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
            const float unit_scale = kLog2e / sqrtf((float)hd);
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
            const uint32_t word = d0 / 8, col = 2 * (s % 4);
            __half* dst = reinterpret_cast<__half*>(qf) + (d0 / 4) % 2;
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
            if (lane == 0) {
                int32_t limit = 0x7fffffff;  // past the last slot: nothing of it is written
                if (live) {
                    const uint32_t pos = p.step[row].position;
                    limit = pos < p.c.seq ? (int32_t)pos : -1;
                }
                slots[s] = Slot{16777216.0f / up, sum, first * (-8.0f / 16777216.0f),
                                rest * (-8.0f / 16777216.0f), limit};
            }
        }
        team_sync<TEAM>();
        float qscale[NT], qsum[NT], qmid[NT][2];  // of slot c (+ 4 nt)
        int32_t limit[NT], lowest = 0x7fffffff;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const Slot& q = slots[c + 4 * nt];
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
        // Weights are w = 2^(score - M). M is the largest score + log2 step of V so far, less 9,
        // moved when a w x step reaches 2^11: as for the queries, its whole number is one operand
        // column, exact in the sums, and the rest the other.
        float o[NT][2 * W][4], l[NT], pm[NT], M[NT], cap[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            l[nt] = pm[nt] = M[nt] = 0.0f;
            cap[nt] = -1.0f;  // no position yet: any moves M
#pragma unroll
            for (int i = 0; i < 2 * W; i++) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f;
        }
        for (; t < t_end; t += TILE) {
            float acc[2][NT][4];
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    acc[i][nt][0] = acc[i][nt][2] = qmid[nt][0];
                    acc[i][nt][1] = acc[i][nt][3] = qmid[nt][1];
                }
#pragma unroll
            for (int w = 0; w < W; w++) {
                uint2 b[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int h = 0; h < 2; h++) b[nt][h] = qf[(nt * W + w) * 2 + h][lane];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const uint32_t x0 = kw[i][0][w], x1 = kw[i][1][w];
                    const uint32_t y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
                        mma16816(acc[i][nt], x0 & M0, x1 & M0, x0 & M1, x1 & M1, b[nt][0].x,
                                 b[nt][0].y);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
                        mma16816(acc[i][nt], y0 & M0, y1 & M0, y0 & M1, y1 & M1, b[nt][1].x,
                                 b[nt][1].y);
                }
            }
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
                        x = fmaf(acc[i / 2][nt][2 * (i % 2) + 1], sq, x);
                        x = fmaf(fmaf(8.0f, step, bf16hi(ks[i])), qsum[nt], x);
                        const bool out = masked.value && (int32_t)(t + 4 * r + i) > limit[nt];
                        sc[nt][i] = out ? -INFINITY : x;
                        w[nt][i] = ex2(sc[nt][i]);
                        ws[nt][i] = out ? 0.0f : w[nt][i] * bf16lo(vs[i]);
                    }
                    over |= fmaxf(fmaxf(ws[nt][0], ws[nt][1]), fmaxf(ws[nt][2], ws[nt][3])) > cap[nt];
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
                        // a step below 2^-90 counts as that: its weight must stay finite
                        const int e = (int)(vs[i] << 16 >> 23) - 127;
                        top = fmaxf(top, sc[nt][i] + (float)max(e, -90));
                    }
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1)
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    if (top > (cap[nt] < 0.0f ? -INFINITY : 9.0f)) {
                        const float to = M[nt] + (top - 9.0f), a = ex2(M[nt] - to);
                        M[nt] = to;
                        if (cap[nt] > 0.0f) {
                            l[nt] *= a;
                            pm[nt] *= a;
#pragma unroll
                            for (int i = 0; i < 2 * W; i++) {
                                o[nt][i][0] *= a; o[nt][i][1] *= a;
                                o[nt][i][2] *= a; o[nt][i][3] *= a;
                            }
                        }
                        cap[nt] = 2048.0f;
                    }
                }
                weigh(std::true_type());
            }
            if (t + TILE < t_end) load_keys(t + TILE);
            uint32_t pb[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    l[nt] += w[nt][i];
                    if (!masked || (int32_t)(t + 4 * r + i) <= limit[nt])
                        pm[nt] = fmaf(w[nt][i], bf16hi(vs[i]), pm[nt]);
                    // the nearest whole number, by way of 1.5 2^23
                    const float first = (ws[nt][i] + 12582912.0f) - 12582912.0f;
                    const __half2 two = __floats2half2_rn(first, ws[nt][i] - first);
                    pb[nt][i] = transpose8(*reinterpret_cast<const uint32_t*>(&two));
                }
            }
            // Sums of 32 positions start from zero and are added to the running ones here: the
            // unit's own addition cuts off, and over a long chain of positive terms that shows
            // (1.4e-5 at 128k positions).
#pragma unroll
            for (int k = 0; k < W; k++) {
                uint32_t y[2][2], z[2][2];
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        y[i][h] = pair_units<W>(vw[i][h][0], vw[i][h][1], k);
                        z[i][h] = y[i][h] >> 8;
                    }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float a[2][4] = {};
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        mma16816(a[0], y[i][0] & M0, y[i][0] & M1, y[i][1] & M0, y[i][1] & M1,
                                 pb[nt][2 * i], pb[nt][2 * i + 1]);
                        mma16816(a[1], z[i][0] & M0, z[i][0] & M1, z[i][1] & M0, z[i][1] & M1,
                                 pb[nt][2 * i], pb[nt][2 * i + 1]);
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int x = 0; x < 4; x++) o[nt][2 * k + h][x] += a[h][x];
                }
            }
            if (t + TILE < t_end) load_values(t + TILE);
        }

        // ---- the warps' parts joined -----------------------------------------------------------
        if constexpr (TEAM == 1) __syncwarp();  // all lanes are done with the queries
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) {
                l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], s);
                pm[nt] += __shfl_xor_sync(0xffffffffu, pm[nt], s);
            }
            if (r == 0) {
                // no positions: no part (a sum that is NaN is one)
                sm[mate][c + 4 * nt] = l[nt] == 0.0f ? -INFINITY : M[nt];
                sl[mate][c + 4 * nt] = l[nt];
            }
#pragma unroll
            for (int i = 0; i < 2 * W; i++) {
                const uint32_t d = (r * W + i / 2) * 4 + 2 * (i % 2);
                *reinterpret_cast<float2*>(&so[mate][c + 4 * nt][d]) =
                    make_float2(fmaf(o[nt][i][0] + o[nt][i][1], 16777216.0f, pm[nt]),
                                fmaf(o[nt][i][2] + o[nt][i][3], 1048576.0f, pm[nt]));
            }
        }
        team_sync<TEAM>();
        float *jm = s_jm[crew], *jl = s_jl[crew];
        if (tt < S) {
            float J = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = 0; w < TEAM; w++) J = fmaxf(J, sm[w][tt]);
#pragma unroll
            for (int w = 0; w < TEAM; w++) {
                const float a = sm[w][tt] == -INFINITY ? 0.0f : ex2(sm[w][tt] - J);
                L = fmaf(sl[w][tt], a, L);
                sm[w][tt] = a;
            }
            jm[tt] = J;
            jl[tt] = L;
        }
        team_sync<TEAM>();
        const bool whole = begin <= span.at && span.until <= end;
        // a unit that began in an earlier stretch is this team's first part, else its last
        float* mine = p.part + (uint64_t)(2 * team + (begin <= span.at)) * PART;
        for (uint32_t i = tt; i < S * HP / 4; i += TT) {
            const uint32_t s = i * 4 / HP, d = i * 4 % HP;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < TEAM; w++) {
                const float4 v = *reinterpret_cast<const float4*>(&so[w][s][d]);
                const float a = sm[w][s];
                x.x = fmaf(v.x, a, x.x);
                x.y = fmaf(v.y, a, x.y);
                x.z = fmaf(v.z, a, x.z);
                x.w = fmaf(v.w, a, x.w);
            }
            if (whole) unit.write(i, x, jl[s]);
            else __stcg(reinterpret_cast<float4*>(mine) + i, x);
        }
        if (!whole) {
            if (tt < S) {
                __stcg(mine + S * HP + tt, jm[tt]);
                __stcg(mine + S * HP + S + tt, jl[tt]);
            }
            team_sync<TEAM>();  // the team's part is written; its first thread publishes it
            if (tt == 0) {
                // teams first .. last meet this unit; the last to arrive joins their parts, after
                // its stretch: up to two units, those at the stretch's ends
                const uint32_t first = line.team_of(span.at);
                const uint32_t parts = line.team_of(span.until - 1) - first + 1;
                uint32_t* ticket = p.tickets + (uint64_t)unit.item * p.per_item + span.nth;
                if (arrive(ticket) == parts - 1) {
                    *ticket = 0;
                    s_job[crew][jobs++] = Job{unit.item, unit.kvh, unit.sub, first, parts};
                }
            }
        }
        at = min(end, span.until);
        team_sync<TEAM>();  // the next unit reuses the shared arrays
    }
    if (tt == 0) s_jobs[crew] = jobs;
    team_sync<TEAM>();
    for (uint32_t k = 0; k < s_jobs[crew]; k++) {
        const Job& job = s_job[crew][k];
        join_parts<W, S, TEAM>(Unit<W, S, OT>{p, job.item, job.kvh, job.sub}, job.first, job.parts,
                               tt, reinterpret_cast<float4*>(so), sm, sl);
        team_sync<TEAM>();
    }
}

template <int W, int NT, int TEAM, typename OT>
void record_one(ab_scheme* s, Kv4AttnParams p, uint32_t grid) {
    constexpr uint32_t S = 4 * NT, PART = S * (32 * W + 2);
    auto* kernel = kv4_attention_kernel<W, NT, TEAM, OT>;
    const uint64_t units = (uint64_t)p.items * p.per_item;
    const uint64_t tiles = units * ((p.c.seq + TEAM * kTurn - 1) / (TEAM * kTurn));
    if (tiles >> 31) invalid("kv4_attention: too much work for one call");
    grid = (uint32_t)std::min<uint64_t>(grid, (tiles * TEAM + kWarps - 1) / kWarps);
    const uint64_t part_bytes = (uint64_t)grid * (kWarps / TEAM) * 2 * PART * 4;
    unsigned char* scratch = nullptr;
    s->rt->activate();
    cuda_check(cudaMalloc((void**)&scratch, part_bytes + units * 4), "cudaMalloc");
    s->owned.push_back(scratch);
    cuda_check(cudaMemset(scratch + part_bytes, 0, units * 4), "clear tickets");
    p.part = (float*)scratch;
    p.tickets = (uint32_t*)(scratch + part_bytes);
    s->add("kv4_attention", [=](cudaStream_t stream) {
        return launch(stream, dim3(grid), dim3(kThreads), 0, true, kernel, p);
    });
}

template <int W, int NT>
void record_slots(ab_scheme* s, const Kv4AttnParams& p, int32_t out_dtype) {
    // one wave; a warp to a team where each unit then meets about eight teams or fewer
    const uint32_t grid = (uint32_t)s->rt->sm_count * (NT == 1 ? 2 : 1);
    const bool solo = (uint64_t)p.items * p.per_item >= grid;
    if (out_dtype == AB_F32)
        solo ? record_one<W, NT, 1, float>(s, p, grid) : record_one<W, NT, 8, float>(s, p, grid);
    else
        solo ? record_one<W, NT, 1, bf16>(s, p, grid) : record_one<W, NT, 8, bf16>(s, p, grid);
}

template <int W>
void record_width(ab_scheme* s, Kv4AttnParams p, int32_t out_dtype) {
    // four query slots a unit where a kv head has no more, else eight
    p.shared = p.c.row_stride == 0 && p.rows > 1;
    const uint64_t slots = p.shared ? (uint64_t)p.rows * p.group : p.group;
    const uint32_t S = slots <= 4 ? 4 : 8;
    const uint32_t blocks = (uint32_t)((slots + S - 1) / S);
    p.items = p.shared ? blocks : p.rows;
    p.per_item = p.c.kv_heads * (p.shared ? 1 : blocks);
    if (S == 4) record_slots<W, 1>(s, p, out_dtype);
    else record_slots<W, 2>(s, p, out_dtype);
}

}  // namespace

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
        Kv4AttnParams p = {};
        p.c = kv4_operands(*cache, rows, kv, head);
        if (numel(out) != (uint64_t)rows * heads * head)
            invalid("parameter `out`: expected " +
                    std::to_string((uint64_t)rows * heads * head) +
                    " elements ([batch, heads * head]), got " + shape_str(out));
        expect_step(step, rows);
        if ((uint64_t)rows * heads > 1u << 30) invalid("parameter `q`: too many rows");
        if (p.c.seq > 0x7fffff00u) invalid("parameter `cache.key_codes`: seq exceeds 2^31 - 256");
        if ((uintptr_t)q.data % 4 || (uintptr_t)out.data % dtype_size(out.dtype))
            invalid("parameter `q` / `out`: not aligned to its elements");
        if (!s->rt)
            fail(AB_ERR_ARGUMENT, "kv4_attention: the scheme needs a runtime (it allocates the "
                                  "split scratch)");
        p.q = (const float*)q.data;
        p.out = out.data;
        p.rows = rows;
        p.heads = heads;
        p.group = heads / kv;
        p.qvec = head % 4 == 0 && (uintptr_t)q.data % 16 == 0;
        p.svec = p.c.seq % 4 == 0 &&
                 ((uintptr_t)p.c.scales[0] | (uintptr_t)p.c.scales[1]) % 16 == 0;
        p.ovec = head % 4 == 0 && (uintptr_t)out.data % (4 * dtype_size(out.dtype)) == 0;
        p.step = (const Step*)step.data;
        p.flags = s->rt->flags;
        switch (p.c.words / 4) {
            case 1: record_width<1>(s, p, out.dtype); break;
            case 2: record_width<2>(s, p, out.dtype); break;
            case 3: record_width<3>(s, p, out.dtype); break;
            default: record_width<4>(s, p, out.dtype); break;
        }
    });
}
