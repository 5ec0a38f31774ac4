// Prompt attention over the 4-bit key/value cache on the 5th-generation tensor cores: rows of one
// shared cache (format: kv4.cu), bf16 outputs. 128 query slots (rows x the query heads of one kv
// head) share every position, so the products are matrix products. With m' = m + 8 s,
//     score_t = (s_t (q . (c_t - 8)) + m'_t sum q) / sqrt(head)
//     out = sum_t p_t (s_t (c_t - 8) + m'_t),  p = softmax over positions 0 .. the row's own:
// c - 8 is a whole number, exact in bf16, so the operands made from the cache lose nothing, and s
// and m' enter per position, outside the products.
//
// One block takes 128 slots of a kv head over a run of 128-position tiles, a slot a TMEM lane:
//  - warps 16-19 read a tile's codes (the next tile's are on their way meanwhile), write them as
//    bf16 operands of K and V in the 128-byte-swizzled layout, and the tile's steps and offsets;
//  - warp 20 (one thread) issues tcgen05.mma: S = Q.(K codes)^T into one of two TMEM buffers, a
//    tile ahead, and O += P.(V codes), V being an MN-major operand of the same layout.
//    Q and P are operands in TMEM: from shared memory, each product read 4 KB of them beside the
//    2 or 4 KB of codes, which made shared memory the bound;
//  - warps 0-15, four threads a slot, make scores of S, keep the slot's maximum and sums, write
//    P = p s of V as the next A operand, and rescale O when the maximum grew by more than
//    kRescale since the scale that O is kept in.
// Q and P are bf16 pairs, value and rest (two products each): 16 bits, 2^-18 of a query or a
// weight, far below the rounding of the output. Elements of a word of codes stay in the order that
// unpacking gives (0 4 1 5 2 6 3 7): Q's dims are staged in the same order, O's put right when
// they are written.
//
// Few blocks split their tiles over several (as many as the device holds at once), and no block
// takes more than kMaxTiles; the last one to finish a slot block joins the parts in order.
// Measured, 8 kv heads of 4 query heads, head 128: 256 rows over 2048 positions 35.5 us (the
// mma.sync kernel of kv4_attention.cu takes 80), 1024 over 8192 346 us (867), of which a tile is
// some 2.5 us: the weights' arithmetic, 16384 exponentials and the scales' broadcast reads, in
// phases that all warps pass together; the products are a third of it. With 64-position tiles, P
// beside S instead of in its place, 39 and 422 us; with Q and P in shared memory 43 and 460.
// Starting and joining is about 11 us.
//
// Every wait is bounded; one that runs out raises the device flag, and the block still lets its
// products finish and frees its TMEM.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "kv4.h"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace ab {

namespace {

constexpr uint32_t kRows = 128;      // slots of a block (TMEM lanes)
constexpr uint32_t kTile = 128;      // positions
constexpr uint32_t kStages = 3;      // tiles unpacked at a time
constexpr uint32_t kShare = 4;       // threads of a slot
constexpr uint32_t kCols = kTile / kShare;
constexpr uint32_t kSoftmax = kRows * kShare;  // threads of warps 0-15
constexpr uint32_t kUnpack = 128;              // of warps 16-19
constexpr uint32_t kUnpackWarp = kSoftmax / 32, kMmaWarp = kUnpackWarp + kUnpack / 32;
constexpr uint32_t kThreads = kSoftmax + kUnpack + 32;
// Columns of TMEM: S twice, each replaced by its P (value, rest), O, Q (value, rest).
constexpr uint32_t kTmemCols = 512, kTmemO = 256, kTmemQ = 384;
constexpr uint32_t kMinTiles = 2;    // a part has at least so many
// and at most these: the tensor unit's additions cut off, so a long chain of them sinks (sums of
// equal codes 2.9e-4 low over 131072 positions, 2.9e-3 over 1000000)
constexpr uint32_t kMaxTiles = 1024;
constexpr float kRescale = 11.5f;    // base 2: P stays below 2^kRescale steps of V
constexpr float kLog2e = 1.4426950408889634f;

struct PromptParams {
    const float* q;  // [rows, heads, head]
    bf16* out;       // [rows, heads * head]
    Kv4View c;
    uint32_t rows, heads, group;
    uint32_t splits, even;  // parts of a slot block at most, and without kMaxTiles
    int qvec, ovec;  // 16-byte accesses of q and out
    float* part;     // [slot block, kv head, split][HD + 2][128]
    uint32_t* tickets;
    const Step* step;
    uint32_t* flags;
};

template <int HD>
struct Layout {
    static constexpr uint32_t T = kTile * HD * 2;  // K or V of a tile
    static constexpr uint32_t SCALES_AT = kStages * 2 * T;  // [stage][K, V][s, m'][kTile]
    static constexpr uint32_t RED_AT = SCALES_AT + kStages * 4 * kTile * 4;
    // maxima [2 tiles][kShare][128]; sums of q, of weights, of weights x m' [kShare][128]
    static constexpr uint32_t BYTES = RED_AT + 5 * kShare * kRows * 4;
};

// Byte offset of 16-byte chunk c (0..7) of row r in a block of 128-byte rows with the 128-byte
// swizzle (eight rows are 1024 bytes).
__device__ __forceinline__ uint32_t row_chunk(uint32_t r, uint32_t c) {
    return (r / 8) * 1024 + (r % 8) * 128 + ((c ^ (r % 8)) * 16);
}
__device__ __forceinline__ void put(uint32_t at, const uint32_t (&w)[4]) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]),
                 "r"(w[2]), "r"(w[3])
                 : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Two floats at a time.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
// Two floats as a bf16 pair and the pair of what rounding left.
__device__ __forceinline__ void split(float a, float b, uint32_t* value, uint32_t* rest) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    *value = *reinterpret_cast<const uint32_t*>(&h);
    const float2 left = fma2(make_float2(bf16lo(*value), bf16hi(*value)), make_float2(-1.0f, -1.0f),
                             make_float2(a, b));
    const __nv_bfloat162 l = __floats2bfloat162_rn(left.x, left.y);
    *rest = *reinterpret_cast<const uint32_t*>(&l);
}
// Codes of a word less 8, as bf16: elements 0 4 1 5 2 6 3 7. A code stands in the low bits of a
// bf16 whose units these are, 128 + c.
__device__ __forceinline__ void unpack(uint32_t word, uint32_t (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t x = (word >> (4 * j) & 0x000f000fu) | 0x43004300u;
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(v[j]) : "r"(x), "r"(0x43084308u));
    }
}
// Not the non-coherent path: the cache's writer may be the grid before this one.
__device__ __forceinline__ uint4 ld16(const uint32_t* p) {
    uint4 r;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p));
    return r;
}
// Asynchronous copy of 16 bytes, or zeros (size 0, nothing is read).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t size) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size)
                 : "memory");
}
__device__ __forceinline__ void copies_wait_all() {
    asm volatile("cp.async.wait_all;" ::: "memory");
}
// Sixteen dims from d on of an output row.
__device__ __forceinline__ void put_out(const PromptParams& p, uint64_t orow, uint32_t d,
                                        const float (&y)[16]) {
    bf16* to = p.out + orow * p.c.head + d;
#pragma unroll
    for (uint32_t k = 0; k < 16; k += 8) {
        if (p.ovec) {
            if (d + k >= p.c.head) continue;
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(y[k + 2 * j], y[k + 2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
            *reinterpret_cast<uint4*>(to + k) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (uint32_t j = k; j < k + 8; j++)
                if (d + j < p.c.head) to[j] = __float2bfloat16_rn(y[j]);
        }
    }
}
// Barrier of the threads that share 32 slots, with the AND of a predicate over them.
__device__ __forceinline__ bool share_sync_and(uint32_t warp, bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
        "bar.red.and.pred p, %2, %3, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)v), "r"(1 + warp % 4), "n"(32 * kShare)
        : "memory");
    return r != 0;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    kv4_prompt_kernel(const __grid_constant__ PromptParams p) {
    using LY = Layout<HD>;
    constexpr uint32_t BOX = HD / 64;  // 64-dim blocks of a row
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full[kStages], empty[kStages], s_full[2], p_full[2], pv_done[2],
        done;
    __shared__ uint32_t s_tmem, s_most[4];
    __shared__ int s_fail, s_last;
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t base = smem_u32(smem);
    float* red = reinterpret_cast<float*>(smem + LY::RED_AT);
    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const uint32_t kvh = blockIdx.y, slot = blockIdx.x * kRows + tid % kRows;

    pdl_wait();
    if (blockIdx.z >= p.even) {  // these parts exist where the others are full
        bool some = false;
        if (tid < kRows && slot / p.group < p.rows) {
            const uint32_t pos = p.step[slot / p.group].position;
            some = pos < p.c.seq && pos / (kTile * kMaxTiles) >= blockIdx.z;
        }
        if (!__syncthreads_or(some)) return;
    }
    // The queries, for now in the room of the later stages: whole rows a few lanes each (a row a
    // thread, read where it is used, took 3 us).
    float* staged = reinterpret_cast<float*>(smem + 2 * LY::T);
    constexpr uint32_t STRIDE = HD + 4;
    static_assert(kRows * STRIDE * 4 <= (kStages - 1) * 2 * LY::T);
    if (tid < kSoftmax) {
#pragma unroll
        for (uint32_t i = tid; i < kRows * HD / 4; i += kSoftmax) {
            const uint32_t d = i % (HD / 4) * 4, sl = blockIdx.x * kRows + i / (HD / 4);
            const uint32_t in = sl / p.group;
            float* to = staged + i / (HD / 4) * STRIDE + d;
            const bool some = in < p.rows && d < p.c.head;
            const float* from = p.q;
            if (some)
                from += ((uint64_t)in * p.heads + kvh * p.group + sl % p.group) * p.c.head + d;
            if (p.qvec) {
                copy16(smem_u32(to), from, some ? 16 : 0);
            } else {
#pragma unroll
                for (uint32_t k = 0; k < 4; k++) to[k] = some && d + k < p.c.head ? from[k] : 0.0f;
            }
        }
        copies_wait_all();
    }
    // the slot's row, head and last position; each of its threads needs them
    const uint32_t row = slot / p.group;
    const bool live = tid < kSoftmax && row < p.rows;
    int32_t limit = -1;
    if (live) {
        const uint32_t pos = p.step[row].position;
        if (pos < p.c.seq) limit = (int32_t)pos;
        else if (kvh == 0 && blockIdx.z == 0) atomicOr(p.flags, kFlagPositionRange);
    }
    const uint64_t orow = (uint64_t)row * p.heads + kvh * p.group + slot % p.group;
    if (warp < 4) {
        const uint32_t most = __reduce_max_sync(0xffffffffu, (uint32_t)(limit + 1));
        if (lane == 0) s_most[warp] = most;
    }
    __syncthreads();
    const uint32_t until = max(max(s_most[0], s_most[1]), max(s_most[2], s_most[3]));
    // the block's share of the tiles
    const uint32_t all = (until + kTile - 1) / kTile;
    const uint32_t each = min(kMaxTiles, max(kMinTiles, (all + p.even - 1) / p.even));
    const uint32_t parts = max(1u, (all + each - 1) / each);
    if (blockIdx.z >= parts) return;
    const uint32_t t_lo = blockIdx.z * each;
    const uint32_t n = min(all, t_lo + each) - t_lo;  // 0 where no row has a position

    if (tid == 0) {
        for (uint32_t i = 0; i < kStages; i++) {
            mbar_init(smem_u32(&full[i]), kUnpack);
            mbar_init(smem_u32(&empty[i]), 1);
        }
        for (uint32_t i = 0; i < 2; i++) {
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&p_full[i]), kSoftmax);
            mbar_init(smem_u32(&pv_done[i]), 1);
        }
        mbar_init(smem_u32(&done), 1);
        fence_barrier_init();
        s_fail = 0;
    }
    if (warp == 0) tmem_alloc(smem_u32(&s_tmem), kTmemCols);
    // a tile's codes, a position a thread of the warps that unpack; the first are on their way
    // while the queries are staged
    const uint32_t line = tid % kUnpack;
    const uint64_t head0 = (uint64_t)kvh * p.c.seq;
    const uint32_t chunks = p.c.words / 4;
    struct Raw {
        uint4 w[2][2 * BOX];  // of K and V, 32 dims each
        uint32_t sc[2];
    };
    auto read = [&](uint32_t tile, Raw& raw) {
        const uint32_t pos = (t_lo + tile) * kTile + line;
        const bool in = tile < n && pos < until;
#pragma unroll
        for (int x = 0; x < 2; x++) {
#pragma unroll
            for (uint32_t c = 0; c < 2 * BOX; c++) {
                raw.w[x][c] = make_uint4(0, 0, 0, 0);
                if (in && c < chunks)
                    raw.w[x][c] = ld16(p.c.codes[x] + (head0 + pos) * p.c.words + 4 * c);
            }
            raw.sc[x] = 0;
            if (in) raw.sc[x] = __ldcg(p.c.scales[x] + head0 + pos);
        }
    };
    Raw raw;
    if (warp >= kUnpackWarp && warp < kMmaWarp) read(0, raw);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const uint32_t mine = tmem + ((warp % 4 * 32) << 16);  // this warp's lanes
    const uint32_t r = tid % kRows, nth = tid / kRows;      // of the threads of slots
    if (tid < kSoftmax) {
        // the slot's queries times log2(e) / sqrt(head): this thread's dims
        const float by = kLog2e / sqrtf((float)p.c.head);
        float sum = 0.0f;
#pragma unroll
        for (uint32_t j = 0; j < HD / (16 * kShare); j++) {
            uint32_t value[8], rest[8];
#pragma unroll
            for (uint32_t e = 0; e < 2; e++) {
                const float* q = staged + r * STRIDE + nth * (HD / kShare) + 16 * j + 8 * e;
                float v[8];
#pragma unroll
                for (uint32_t k = 0; k < 8; k += 4) {
                    const float4 x = *reinterpret_cast<const float4*>(q + k);
                    v[k] = x.x * by;
                    v[k + 1] = x.y * by;
                    v[k + 2] = x.z * by;
                    v[k + 3] = x.w * by;
                    sum += (v[k] + v[k + 1]) + (v[k + 2] + v[k + 3]);
                }
#pragma unroll
                for (int k = 0; k < 4; k++)
                    split(v[k], v[k + 4], &value[4 * e + k], &rest[4 * e + k]);
            }
            const uint32_t at = mine + kTmemQ + nth * (HD / (2 * kShare)) + 8 * j;
            tmem_st8(at, value);
            tmem_st8(at + HD / 2, rest);
        }
        red[(2 * kShare + nth) * kRows + r] = sum;
        tmem_wait_st();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();

    float m_ref = -INFINITY, l = 0.0f, pm = 0.0f;
    if (warp >= kUnpackWarp && warp < kMmaWarp) {
        // ---- codes to operands: a position a thread ----
        auto write = [&](uint32_t i, const Raw& raw) {
            const uint32_t s = i % kStages;
            if (i >= kStages && !mbar_wait_bounded(smem_u32(&empty[s]), (i / kStages - 1) & 1,
                                                   p.flags))
                return false;
            const uint32_t to = base + s * 2 * LY::T;
            float* scales = reinterpret_cast<float*>(smem + LY::SCALES_AT) + s * (4 * kTile) + line;
#pragma unroll
            for (int x = 0; x < 2; x++) {
#pragma unroll
                for (uint32_t c = 0; c < 2 * BOX; c++) {
                    const uint4& w = raw.w[x][c];
                    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (uint32_t k = 0; k < 4; k++) {
                        uint32_t v[4];
                        unpack(word[k], v);
                        put(to + x * LY::T + c / 2 * (kTile * 128) +
                                row_chunk(line, c % 2 * 4 + k),
                            v);
                    }
                }
                scales[2 * x * kTile] = bf16lo(raw.sc[x]);
                scales[(2 * x + 1) * kTile] = fmaf(8.0f, bf16lo(raw.sc[x]), bf16hi(raw.sc[x]));
            }
            fence_proxy_async_smem();
            mbar_arrive(smem_u32(&full[s]));
            return true;
        };
        bool ok = true;
        for (uint32_t i = 0; i < n && ok; i++) {
            ok = write(i, raw);
            read(i + 1, raw);
        }
        if (!ok) s_fail = 1;
    } else if (warp == kMmaWarp) {
        if (lane == 0 && n > 0) {
            const uint32_t idesc_s = tc_idesc_bf16(kRows, kTile);
            const uint32_t idesc_o = tc_idesc_bf16(kRows, HD) | kIdescBMajorMN;
            auto scores = [&](uint32_t i) {
                const uint32_t s = i % kStages;
                if (!mbar_wait_bounded(smem_u32(&full[s]), (i / kStages) & 1, p.flags))
                    return false;
                // its buffer holds the P before the last until that has been multiplied
                if (i >= 2 &&
                    !mbar_wait_bounded(smem_u32(&pv_done[i % 2]), (i / 2 - 1) & 1, p.flags))
                    return false;
                tc_fence_after();
                const uint32_t k_at = base + s * 2 * LY::T;
                const uint32_t d = tmem + (i % 2) * kTile;
#pragma unroll
                for (uint32_t b = 0; b < BOX; b++) {
                    const uint64_t kd = sw128_desc(k_at + b * (kTile * 128));
#pragma unroll
                    for (uint32_t k = 0; k < 4; k++) {
                        const uint32_t q = tmem + kTmemQ + 32 * b + 8 * k;
                        tc_mma_bf16_ta(d, q, kd + 2 * k, idesc_s, (b | k) != 0);
                        tc_mma_bf16_ta(d, q + HD / 2, kd + 2 * k, idesc_s, 1);
                    }
                }
                tc_commit(smem_u32(&s_full[i % 2]));
                return true;
            };
            bool ok = scores(0);
            for (uint32_t i = 0; i < n && ok; i++) {
                if (i + 1 < n && !scores(i + 1)) {
                    ok = false;
                    break;
                }
                if (!mbar_wait_bounded(smem_u32(&p_full[i % 2]), (i / 2) & 1, p.flags)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t v_at = base + (i % kStages * 2 + 1) * LY::T;
                const uint32_t w = tmem + i % 2 * kTile;
#pragma unroll
                for (uint32_t k = 0; k < kTile / 16; k++) {
                    const uint64_t vd = sw128_desc_mn(v_at + k * 16 * 128, kTile * 128);
                    tc_mma_bf16_ta(tmem + kTmemO, w + 8 * k, vd, idesc_o, (i | k) != 0);
                    tc_mma_bf16_ta(tmem + kTmemO, w + kTile / 2 + 8 * k, vd, idesc_o, 1);
                }
                tc_commit(smem_u32(&pv_done[i % 2]));
                tc_commit(smem_u32(&empty[i % kStages]));
            }
            if (!ok) s_fail = 1;
        }
        if (lane == 0) tc_commit(smem_u32(&done));  // all that this thread issued
    } else if (tid < kSoftmax) {
        // ---- weights: thread `nth` of a slot has columns kCols nth .. of S, HD / kShare nth .. of
        // O ----
        float qs = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < kShare; k++) qs += red[(2 * kShare + k) * kRows + r];
        const float2 qsum = make_float2(qs, qs);
        bool ok = true, failed = false;
        for (uint32_t i = 0; i < n; i++) {
            bool w = mbar_wait_bounded(smem_u32(&s_full[i % 2]), (i / 2) & 1, p.flags);
            w = mbar_wait_bounded(smem_u32(&full[i % kStages]), (i / kStages) & 1, p.flags) && w;
            __syncwarp();
            tc_fence_after();
            const float4* scales = reinterpret_cast<const float4*>(smem + LY::SCALES_AT) +
                                   i % kStages * kTile + nth * (kCols / 4);
            float2 x[kCols / 2];
#pragma unroll
            for (uint32_t c = 0; c < kCols / 16; c++) {
                float xs[16];
                tmem_ld16(mine + (i % 2) * kTile + nth * kCols + 16 * c, xs);
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) {
                    const float4 ks = scales[4 * c + j], km = scales[kTile / 4 + 4 * c + j];
                    x[8 * c + 2 * j] =
                        fma2(make_float2(xs[4 * j], xs[4 * j + 1]), make_float2(ks.x, ks.y),
                             mul2(qsum, make_float2(km.x, km.y)));
                    x[8 * c + 2 * j + 1] =
                        fma2(make_float2(xs[4 * j + 2], xs[4 * j + 3]), make_float2(ks.z, ks.w),
                             mul2(qsum, make_float2(km.z, km.w)));
                }
            }
            tc_fence_before();
            // columns 0 .. seen are attended over; what the others hold is not used, NaN or not
            const int32_t seen = limit - (int32_t)((t_lo + i) * kTile + nth * kCols);
            if (seen < (int32_t)kCols - 1) {
#pragma unroll
                for (int j = 0; j < (int)kCols / 2; j++) {
                    if (2 * j > seen) x[j].x = -INFINITY;
                    if (2 * j + 1 > seen) x[j].y = -INFINITY;
                }
            }
            float most = fmaxf(x[0].x, x[0].y);
#pragma unroll
            for (uint32_t j = 1; j < kCols / 2; j++) most = fmaxf(fmaxf(most, x[j].x), x[j].y);
            float* maxima = red + (i & 1) * (kShare * kRows) + r;
            maxima[nth * kRows] = most;
            ok = share_sync_and(warp, w && !failed);
            if (!ok) break;
            tc_fence_after();  // the slot's S has been read: P may take its place
#pragma unroll
            for (uint32_t k = 0; k < kShare; k++) most = fmaxf(most, maxima[k * kRows]);
            float alpha = 1.0f;
            bool rescale = false;
            if (most != -INFINITY && (m_ref == -INFINITY || most > m_ref + kRescale)) {
                if (m_ref != -INFINITY) {
                    alpha = ex2(m_ref - most);
                    rescale = true;
                }
                m_ref = most;
            }
            const float m0 = m_ref == -INFINITY ? 0.0f : -m_ref;  // nothing seen: weights of 0
            const float2 m2 = make_float2(m0, m0);
            float2 sum = make_float2(0.0f, 0.0f), off = sum;
            auto weigh = [&](auto masked) {
#pragma unroll
                for (int j = 0; j < (int)kCols / 4; j++) {
                    const float4 vs = scales[2 * (kTile / 4) + j], vm = scales[3 * (kTile / 4) + j];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float2 s2 = e ? make_float2(vs.z, vs.w) : make_float2(vs.x, vs.y);
                        float2 o2 = e ? make_float2(vm.z, vm.w) : make_float2(vm.x, vm.y);
                        if constexpr (decltype(masked)::value) {
                            if (4 * j + 2 * e > seen) s2.x = o2.x = 0.0f;
                            if (4 * j + 2 * e + 1 > seen) s2.y = o2.y = 0.0f;
                        }
                        const float2 y = add2(x[2 * j + e], m2);
                        const float2 a = make_float2(ex2(y.x), ex2(y.y));
                        sum = add2(sum, a);
                        off = fma2(a, o2, off);
                        x[2 * j + e] = mul2(a, s2);
                    }
                }
            };
            if (seen < (int32_t)kCols - 1) weigh(std::true_type());
            else weigh(std::false_type());
            l = fmaf(l, alpha, sum.x + sum.y);
            pm = fmaf(pm, alpha, off.x + off.y);
            // O is at rest once the tile before is in it
            if (i >= 1 && __any_sync(0xffffffffu, rescale)) {
                if (!mbar_wait_bounded(smem_u32(&pv_done[(i - 1) % 2]), ((i - 1) / 2) & 1, p.flags))
                    failed = true;
                __syncwarp();
                tc_fence_after();
#pragma unroll
                for (uint32_t c = 0; c < HD / (16 * kShare); c++) {
                    float o[16];
                    const uint32_t at = mine + kTmemO + nth * (HD / kShare) + 16 * c;
                    tmem_ld16(at, o);
#pragma unroll
                    for (int k = 0; k < 16; k++) o[k] *= alpha;
                    tmem_st16(at, o);
                }
            }
#pragma unroll
            for (uint32_t c = 0; c < kCols / 2; c += 8) {
                uint32_t value[8], rest[8];
#pragma unroll
                for (int k = 0; k < 8; k++) split(x[c + k].x, x[c + k].y, &value[k], &rest[k]);
                const uint32_t at = mine + i % 2 * kTile + nth * (kCols / 2) + c;
                tmem_st8(at, value);
                tmem_st8(at + kTile / 2, rest);
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(smem_u32(&p_full[i % 2]));
        }
        bool w = true;
        if (ok && n > 0) w = mbar_wait_bounded(smem_u32(&pv_done[(n - 1) % 2]), ((n - 1) / 2) & 1, p.flags);
        red[(3 * kShare + nth) * kRows + r] = l;
        red[(4 * kShare + nth) * kRows + r] = pm;
        ok = share_sync_and(warp, ok && w && !failed);
        l = pm = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < kShare; k++) {
            l += red[(3 * kShare + k) * kRows + r];
            pm += red[(4 * kShare + k) * kRows + r];
        }
        if (!ok) s_fail = 1;
        tc_fence_after();
        float* part = p.part + (((uint64_t)blockIdx.x * p.c.kv_heads + kvh) * p.splits +
                                blockIdx.z) * ((HD + 2) * kRows);
        const float by = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (uint32_t c = 0; c < HD / (16 * kShare); c++) {
            const uint32_t d = nth * (HD / kShare) + 16 * c;
            float o[16];
#pragma unroll
            for (int k = 0; k < 16; k++) o[k] = 0.0f;
            if (ok && n > 0) tmem_ld16(mine + kTmemO + d, o);
            if (parts == 1) {
                float y[16];
#pragma unroll
                for (int k = 0; k < 16; k++)
                    y[k] = (o[k / 8 * 8 + 2 * (k % 4) + k % 8 / 4] + pm) * by;
                if (live) put_out(p, orow, d, y);
            } else {
#pragma unroll
                for (int k = 0; k < 16; k += 4) {
                    const float* at = o + k / 8 * 8 + k % 8 / 4;
                    __stcg(reinterpret_cast<float4*>(part) + (d + k) / 4 * kRows + r,
                           make_float4(at[0] + pm, at[2] + pm, at[4] + pm, at[6] + pm));
                }
            }
        }
        if (parts > 1 && nth == 0) {
            __stcg(part + HD * kRows + r, m_ref);
            __stcg(part + (HD + 1) * kRows + r, l);
        }
    }
    __syncthreads();
    if (parts > 1) {
        if (tid == 0) {
            uint32_t* ticket = p.tickets + (uint64_t)blockIdx.x * p.c.kv_heads + kvh;
            const bool last = kv4_arrive(ticket) == parts - 1;
            if (last) *ticket = 0;
            s_last = last;
        }
        __syncthreads();
        if (s_last && tid < kSoftmax) {
            const float* part = p.part + ((uint64_t)blockIdx.x * p.c.kv_heads + kvh) * p.splits *
                                             ((HD + 2) * kRows);
            float M = -INFINITY, L = 0.0f;
            float4 y[HD / (4 * kShare)];
#pragma unroll 4
            for (uint32_t z = 0; z < parts; z++)
                M = fmaxf(M, __ldcg(part + (z * (HD + 2) + HD) * kRows + r));
#pragma unroll
            for (uint32_t k = 0; k < HD / (4 * kShare); k++) y[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (uint32_t z = 0; z < parts; z++) {
                const float* pz = part + z * ((HD + 2) * kRows);
                float4 v[HD / (4 * kShare)];
#pragma unroll
                for (uint32_t k = 0; k < HD / (4 * kShare); k++)
                    v[k] = __ldcg(reinterpret_cast<const float4*>(pz) +
                                  (nth * (HD / (4 * kShare)) + k) * kRows + r);
                const float mz = __ldcg(pz + HD * kRows + r), lz = __ldcg(pz + (HD + 1) * kRows + r);
                const float f = mz == -INFINITY ? 0.0f : ex2(mz - M);
                L = fmaf(lz, f, L);
#pragma unroll
                for (uint32_t k = 0; k < HD / (4 * kShare); k++) {
                    y[k].x = fmaf(v[k].x, f, y[k].x);
                    y[k].y = fmaf(v[k].y, f, y[k].y);
                    y[k].z = fmaf(v[k].z, f, y[k].z);
                    y[k].w = fmaf(v[k].w, f, y[k].w);
                }
            }
            const float by = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
            for (uint32_t c = 0; c < HD / (16 * kShare); c++) {
                float v[16];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    v[4 * k] = y[4 * c + k].x * by;
                    v[4 * k + 1] = y[4 * c + k].y * by;
                    v[4 * k + 2] = y[4 * c + k].z * by;
                    v[4 * k + 3] = y[4 * c + k].w * by;
                }
                if (live) put_out(p, orow, nth * (HD / kShare) + 16 * c, v);
            }
        }
    }
    if (warp == 0) {
        if (lane == 0 && s_fail) atomicOr(p.flags, kFlagWaitTimeout);
        mbar_wait_bounded(smem_u32(&done), 0, p.flags);  // every product has finished
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
    pdl_trigger();
}

template <int HD>
void record_one(ab_scheme* s, const char* label, PromptParams p) {
    auto* kernel = kv4_prompt_kernel<HD>;
    constexpr size_t smem = Layout<HD>::BYTES + 1024;
    static_assert(smem + 512 <= 227 * 1024);
    const uint64_t blocks = ((uint64_t)p.rows * p.group + kRows - 1) / kRows;
    const uint64_t units = blocks * p.c.kv_heads;
    const uint32_t longest = (uint32_t)(((uint64_t)p.c.seq + kTile * kMaxTiles - 1) / (kTile * kMaxTiles));
    p.even = (uint32_t)std::max<uint64_t>(1, s->rt->sm_count / units);
    p.splits = std::max(p.even, longest);
    s->rt->activate();
    cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
               "kv4_attention shared memory");
    kv4_take_scratch(s, p.splits > 1 ? units * p.splits * (HD + 2) * kRows * 4 : 0, units, &p.part,
                     &p.tickets);
    const dim3 grid((unsigned)blocks, p.c.kv_heads, p.splits);
    s->add(label, [=](cudaStream_t stream) {
        return launch(stream, grid, dim3(kThreads), smem, true, kernel, p);
    });
}

}  // namespace

bool record_kv4_prompt_tc(ab_scheme* s, const char* label, const float* q, uint32_t rows,
                          uint32_t heads, const Kv4View& cache, void* out, const Step* step) {
    PromptParams p = {};
    p.q = q;
    p.out = (bf16*)out;
    p.c = cache;
    p.rows = rows;
    p.heads = heads;
    p.group = heads / cache.kv_heads;
    if (cache.row_stride != 0 || cache.kv_heads > 65535) return false;
    p.qvec = cache.head % 4 == 0 && (uintptr_t)q % 16 == 0;
    p.ovec = cache.head % 8 == 0 && (uintptr_t)out % 16 == 0;
    p.step = step;
    p.flags = s->rt->flags;
    if (cache.words <= 8) record_one<64>(s, label, p);
    else record_one<128>(s, label, p);
    return true;
}

}  // namespace ab
