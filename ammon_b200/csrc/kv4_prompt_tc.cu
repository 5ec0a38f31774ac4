// Prompt attention over the 4-bit key/value cache on the 5th-generation tensor cores: rows of one
// shared cache (format: kv4.cu), bf16 outputs. 128 query slots (rows x the query heads of one kv
// head) share every position, so the products are matrix products. With m' = m + 8 s,
//     score_t = (s_t (q . (c_t - 8)) + m'_t sum q) / sqrt(head)
//     out = sum_t p_t (s_t (c_t - 8) + m'_t),  p = softmax over positions 0 .. the row's own:
// c - 8 is a whole number, exact in bf16, so the operands made from the cache lose nothing, and s
// and m' enter per position, outside the products.
//
// One block takes 128 slots of a kv head over a run of 64-position tiles, a slot a TMEM lane:
//  - warps 8-11 read a tile's codes (the next tile's are on their way meanwhile), write them as
//    bf16 operands of K and V in the 128-byte-swizzled layout, and the tile's steps and offsets;
//  - warp 12 (one thread) issues tcgen05.mma: S = Q.(K codes)^T into one of two 64-column TMEM
//    buffers, a tile ahead, and O += P.(V codes), V being an MN-major operand of the same layout;
//  - warps 0-7, two threads a slot, make scores of S, keep the slot's maximum and sums, write
//    P = p s of V as the next A operand, and rescale O when the maximum grew by more than
//    kRescale since the scale that O is kept in.
// Q and P are bf16 pairs, value and rest (two products each): 16 bits, 2^-18 of a query or a
// weight, far below the rounding of the output. Elements of a word of codes stay in the order that
// unpacking gives (0 4 1 5 2 6 3 7): Q's dims are staged in the same order, O's put right when
// they are written.
//
// Few blocks split their tiles over several (as many as the device holds at once); the last one
// to finish a slot block joins the parts in order.
// Every wait is bounded; one that runs out raises the device flag, and the block still lets its
// products finish and frees its TMEM.
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "kv4.h"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace ab {

namespace {

constexpr uint32_t kRows = 128;      // slots of a block (TMEM lanes)
constexpr uint32_t kTile = 64;       // positions
constexpr uint32_t kStages = 3;      // tiles unpacked at a time
constexpr uint32_t kSoftmax = 256;   // threads of warps 0-7
constexpr uint32_t kUnpack = 128;    // of warps 8-11
constexpr uint32_t kThreads = kSoftmax + kUnpack + 32;
constexpr uint32_t kTmemCols = 256;  // S at columns 0 and 64, O from 128
constexpr uint32_t kTmemO = 128;
constexpr uint32_t kMinTiles = 4;    // a part has at least so many
constexpr float kRescale = 11.5f;    // base 2: P stays below 2^kRescale steps of V
constexpr float kLog2e = 1.4426950408889634f;

struct PromptParams {
    const float* q;  // [rows, heads, head]
    bf16* out;       // [rows, heads * head]
    Kv4View c;
    uint32_t rows, heads, group, splits;
    int qvec, ovec;  // 16-byte accesses of q and out
    float* part;     // [slot block, kv head, split][HD + 2][128]
    uint32_t* tickets;
    const Step* step;
    uint32_t* flags;
};

template <int HD>
struct Layout {
    static constexpr uint32_t Q = kRows * HD * 2;     // value, then rest
    static constexpr uint32_t P = kRows * kTile * 2;  // value, then rest
    static constexpr uint32_t T = kTile * HD * 2;     // K or V of a tile
    static constexpr uint32_t P_AT = 2 * Q, KV_AT = P_AT + 2 * P;
    static constexpr uint32_t SCALES_AT = KV_AT + kStages * 2 * T;  // [stage][K, V][64] (s, m')
    static constexpr uint32_t RED_AT = SCALES_AT + kStages * 2 * kTile * 8;
    // maxima [2 tiles][2 halves][128]; sums of q, of weights, of weights x m' [2 halves][128]
    static constexpr uint32_t BYTES = RED_AT + 10 * kRows * 4;
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
// Two floats as a bf16 pair and the pair of what rounding left.
__device__ __forceinline__ void split(float a, float b, uint32_t* value, uint32_t* rest) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    *value = *reinterpret_cast<const uint32_t*>(&h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(a - bf16lo(*value), b - bf16hi(*value));
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
// Barrier of the 64 threads that share 32 slots, with the AND of a predicate over them.
__device__ __forceinline__ bool pair_sync_and(uint32_t warp, bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
        "bar.red.and.pred p, %2, 64, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)v), "r"(1 + warp % 4)
        : "memory");
    return r != 0;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    kv4_prompt_kernel(const __grid_constant__ PromptParams p) {
    using LY = Layout<HD>;
    constexpr uint32_t BOX = HD / 64;  // 64-dim blocks of a row
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full[kStages], empty[kStages], s_full[2], s_free[2], p_full,
        pv_done, done;
    __shared__ uint32_t s_tmem, s_most[4];
    __shared__ int s_fail, s_last;
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t base = smem_u32(smem);
    float* red = reinterpret_cast<float*>(smem + LY::RED_AT);
    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const uint32_t kvh = blockIdx.y, slot = blockIdx.x * kRows + tid % kRows;

    pdl_wait();
    // the slot's row, head and last position; both threads of a slot need them
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
    const uint32_t each = max(kMinTiles, (all + p.splits - 1) / p.splits);
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
            mbar_init(smem_u32(&s_free[i]), kSoftmax);
        }
        mbar_init(smem_u32(&p_full), kSoftmax);
        mbar_init(smem_u32(&pv_done), 1);
        mbar_init(smem_u32(&done), 1);
        fence_barrier_init();
        s_fail = 0;
    }
    if (warp == 0) tmem_alloc(smem_u32(&s_tmem), kTmemCols);
    if (tid < kSoftmax) {
        // the slot's queries times log2(e) / sqrt(head): this half's dims
        const uint32_t r = tid % kRows, half = tid / kRows;
        const float by = kLog2e / sqrtf((float)p.c.head);
        const float* q = p.q + orow * p.c.head;
        float sum = 0.0f;
#pragma unroll
        for (uint32_t j = 0; j < HD / 16; j++) {
            const uint32_t chunk = half * (HD / 16) + j, d = chunk * 8;
            float v[8];
#pragma unroll
            for (uint32_t k = 0; k < 8; k += 4) {
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (limit >= 0 && d + k < p.c.head) {
                    if (p.qvec) {
                        x = *reinterpret_cast<const float4*>(q + d + k);
                    } else {
                        const uint32_t left = p.c.head - d - k;
                        x.x = q[d + k];
                        if (left > 1) x.y = q[d + k + 1];
                        if (left > 2) x.z = q[d + k + 2];
                        if (left > 3) x.w = q[d + k + 3];
                    }
                }
                v[k] = x.x * by;
                v[k + 1] = x.y * by;
                v[k + 2] = x.z * by;
                v[k + 3] = x.w * by;
                sum += (v[k] + v[k + 1]) + (v[k + 2] + v[k + 3]);
            }
            uint32_t value[4], rest[4];
#pragma unroll
            for (int k = 0; k < 4; k++) split(v[k], v[k + 4], &value[k], &rest[k]);
            const uint32_t at = base + chunk / 8 * (kRows * 128) + row_chunk(r, chunk % 8);
            put(at, value);
            put(at + LY::Q, rest);
        }
        red[(4 + half) * kRows + r] = sum;
        fence_proxy_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    float m_ref = -INFINITY, l = 0.0f, pm = 0.0f;
    if (warp >= 8 && warp < 12) {
        // ---- codes to operands: a thread half of a position's chunks (32 dims each) ----
        const uint32_t u = tid - kSoftmax, r = u / 2, odd = u % 2;
        const uint64_t head0 = (uint64_t)kvh * p.c.seq;
        const uint32_t chunks = p.c.words / 4;
        uint4 w[2][BOX];
        uint32_t sc = 0;  // of K (even threads) or V
        auto read = [&](uint32_t tile) {
            const uint32_t pos = (t_lo + tile) * kTile + r;
            const bool in = tile < n && pos < until;
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (uint32_t b = 0; b < BOX; b++) {
                    const uint32_t c = 2 * b + odd;
                    w[x][b] = make_uint4(0, 0, 0, 0);
                    if (in && c < chunks)
                        w[x][b] = ld16(p.c.codes[x] + (head0 + pos) * p.c.words + 4 * c);
                }
            sc = 0;
            if (in) sc = __ldcg(p.c.scales[odd] + head0 + pos);
        };
        read(0);
        for (uint32_t i = 0; i < n; i++) {
            const uint32_t s = i % kStages;
            if (i >= kStages && !mbar_wait_bounded(smem_u32(&empty[s]), (i / kStages - 1) & 1,
                                                   p.flags)) {
                s_fail = 1;
                break;
            }
            const uint32_t to = base + LY::KV_AT + s * 2 * LY::T;
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (uint32_t b = 0; b < BOX; b++) {
                    const uint32_t word[4] = {w[x][b].x, w[x][b].y, w[x][b].z, w[x][b].w};
#pragma unroll
                    for (uint32_t k = 0; k < 4; k++) {
                        uint32_t v[4];
                        unpack(word[k], v);
                        put(to + x * LY::T + b * (kTile * 128) + row_chunk(r, 4 * odd + k), v);
                    }
                }
            float2* scales = reinterpret_cast<float2*>(smem + LY::SCALES_AT) +
                             (s * 2 + odd) * kTile + r;
            *scales = make_float2(bf16lo(sc), fmaf(8.0f, bf16lo(sc), bf16hi(sc)));
            fence_proxy_async_smem();
            mbar_arrive(smem_u32(&full[s]));
            read(i + 1);
        }
    } else if (warp == 12) {
        if (lane == 0 && n > 0) {
            const uint32_t idesc_s = tc_idesc_bf16(kRows, kTile);
            const uint32_t idesc_o = tc_idesc_bf16(kRows, HD) | kIdescBMajorMN;
            auto scores = [&](uint32_t i) {
                const uint32_t s = i % kStages;
                if (!mbar_wait_bounded(smem_u32(&full[s]), (i / kStages) & 1, p.flags))
                    return false;
                // the tile before the last has been read out of this buffer
                if (i >= 2 && !mbar_wait_bounded(smem_u32(&s_free[i % 2]), (i / 2 - 1) & 1, p.flags))
                    return false;
                tc_fence_after();
                const uint32_t k_at = base + LY::KV_AT + s * 2 * LY::T;
                const uint32_t d = tmem + (i % 2) * kTile;
#pragma unroll
                for (uint32_t b = 0; b < BOX; b++) {
                    const uint64_t qv = sw128_desc(base + b * (kRows * 128));
                    const uint64_t qr = sw128_desc(base + LY::Q + b * (kRows * 128));
                    const uint64_t kd = sw128_desc(k_at + b * (kTile * 128));
#pragma unroll
                    for (uint32_t k = 0; k < 4; k++) {
                        tc_mma_bf16(d, qv + 2 * k, kd + 2 * k, idesc_s, (b | k) != 0);
                        tc_mma_bf16(d, qr + 2 * k, kd + 2 * k, idesc_s, 1);
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
                if (!mbar_wait_bounded(smem_u32(&p_full), i & 1, p.flags)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t v_at = base + LY::KV_AT + (i % kStages * 2 + 1) * LY::T;
                const uint64_t pv = sw128_desc(base + LY::P_AT);
                const uint64_t pr = sw128_desc(base + LY::P_AT + LY::P);
#pragma unroll
                for (uint32_t k = 0; k < kTile / 16; k++) {
                    const uint64_t vd = sw128_desc_mn(v_at + k * 16 * 128, kTile * 128);
                    tc_mma_bf16(tmem + kTmemO, pv + 2 * k, vd, idesc_o, (i | k) != 0);
                    tc_mma_bf16(tmem + kTmemO, pr + 2 * k, vd, idesc_o, 1);
                }
                tc_commit(smem_u32(&pv_done));
                tc_commit(smem_u32(&empty[i % kStages]));
            }
            if (!ok) s_fail = 1;
        }
        if (lane == 0) tc_commit(smem_u32(&done));  // all that this thread issued
    } else if (warp < 8) {
        // ---- weights: thread `half` of a slot has columns 32 half .. of S, HD / 2 half .. of O --
        const uint32_t r = tid % kRows, half = tid / kRows;
        const uint32_t mine = tmem + ((warp % 4 * 32) << 16);  // this warp's lanes
        const float qsum = red[4 * kRows + r] + red[5 * kRows + r];
        bool ok = true, failed = false;
        for (uint32_t i = 0; i < n; i++) {
            bool w = mbar_wait_bounded(smem_u32(&s_full[i % 2]), (i / 2) & 1, p.flags);
            w = mbar_wait_bounded(smem_u32(&full[i % kStages]), (i / kStages) & 1, p.flags) && w;
            tc_fence_after();
            float x[32];
            tmem_ld16(mine + (i % 2) * kTile + half * 32, x);
            tmem_ld16(mine + (i % 2) * kTile + half * 32 + 16, x + 16);
            tc_fence_before();
            mbar_arrive(smem_u32(&s_free[i % 2]));
            const float4* ks = reinterpret_cast<const float4*>(smem + LY::SCALES_AT) +
                               i % kStages * kTile + half * 16;
            const float4* vs = ks + kTile / 2;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const float4 k = ks[j];
                x[2 * j] = fmaf(x[2 * j], k.x, qsum * k.y);
                x[2 * j + 1] = fmaf(x[2 * j + 1], k.z, qsum * k.w);
            }
            const int32_t t0 = (int32_t)((t_lo + i) * kTile + half * 32);
            const int32_t seen = limit - t0;  // columns 0 .. seen are attended over
            if (seen < 31) {
#pragma unroll
                for (int j = 0; j < 32; j++)
                    if (j > seen) x[j] = -INFINITY;
            }
            float most = x[0];
#pragma unroll
            for (int j = 1; j < 32; j++) most = fmaxf(most, x[j]);
            red[((i & 1) * 2 + half) * kRows + r] = most;
            ok = pair_sync_and(warp, w && !failed);
            if (!ok) break;
            most = fmaxf(most, red[((i & 1) * 2 + (half ^ 1)) * kRows + r]);
            float alpha = 1.0f;
            bool rescale = false;
            if (most != -INFINITY && (m_ref == -INFINITY || most > m_ref + kRescale)) {
                if (m_ref != -INFINITY) {
                    alpha = ex2(m_ref - most);
                    rescale = true;
                }
                m_ref = most;
            }
            const float m0 = m_ref == -INFINITY ? 0.0f : m_ref;  // nothing seen: weights of 0
            float sum = 0.0f, off = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const float4 v = vs[j];
                const float a = ex2(x[2 * j] - m0), b = ex2(x[2 * j + 1] - m0);
                sum += a + b;
                x[2 * j] = a * v.x;
                x[2 * j + 1] = b * v.z;
                if (seen < 31) {  // what lies past the row's position is not used, NaN or not
                    if (2 * j > seen) x[2 * j] = 0.0f;
                    if (2 * j + 1 > seen) x[2 * j + 1] = 0.0f;
                    off = fmaf(a, 2 * j > seen ? 0.0f : v.y, off);
                    off = fmaf(b, 2 * j + 1 > seen ? 0.0f : v.w, off);
                } else {
                    off = fmaf(a, v.y, off);
                    off = fmaf(b, v.w, off);
                }
            }
            l = fmaf(l, alpha, sum);
            pm = fmaf(pm, alpha, off);
            // P's place and O are free once the tile before is in O
            if (i >= 1 && !mbar_wait_bounded(smem_u32(&pv_done), (i - 1) & 1, p.flags))
                failed = true;
            tc_fence_after();
            if (i >= 1 && __any_sync(0xffffffffu, rescale)) {
#pragma unroll
                for (uint32_t c = 0; c < HD / 32; c++) {
                    float o[16];
                    const uint32_t at = mine + kTmemO + half * (HD / 2) + 16 * c;
                    tmem_ld16(at, o);
#pragma unroll
                    for (int k = 0; k < 16; k++) o[k] *= alpha;
                    tmem_st16(at, o);
                }
                tmem_wait_st();
            }
#pragma unroll
            for (uint32_t c = 0; c < 4; c++) {
                uint32_t value[4], rest[4];
#pragma unroll
                for (int k = 0; k < 4; k++)
                    split(x[8 * c + 2 * k], x[8 * c + 2 * k + 1], &value[k], &rest[k]);
                const uint32_t at = base + LY::P_AT + row_chunk(r, half * 4 + c);
                put(at, value);
                put(at + LY::P, rest);
            }
            fence_proxy_async_smem();
            tc_fence_before();
            mbar_arrive(smem_u32(&p_full));
        }
        bool w = true;
        if (ok && n > 0) w = mbar_wait_bounded(smem_u32(&pv_done), (n - 1) & 1, p.flags);
        red[(6 + half) * kRows + r] = l;
        red[(8 + half) * kRows + r] = pm;
        ok = pair_sync_and(warp, ok && w && !failed);
        l = red[6 * kRows + r] + red[7 * kRows + r];
        pm = red[8 * kRows + r] + red[9 * kRows + r];
        if (!ok) s_fail = 1;
        tc_fence_after();
        float* part = p.part + (((uint64_t)blockIdx.x * p.c.kv_heads + kvh) * p.splits +
                                blockIdx.z) * ((HD + 2) * kRows);
        const float by = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
        for (uint32_t c = 0; c < HD / 32; c++) {
            const uint32_t d = half * (HD / 2) + 16 * c;
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
                for (int k = 0; k < 16; k++)
                    __stcg(part + (d + k) * kRows + r, o[k / 8 * 8 + 2 * (k % 4) + k % 8 / 4] + pm);
            }
        }
        if (parts > 1 && half == 0) {
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
            const uint32_t r = tid % kRows, half = tid / kRows;
            const float* part = p.part + ((uint64_t)blockIdx.x * p.c.kv_heads + kvh) * p.splits *
                                             ((HD + 2) * kRows) + r;
            float M = -INFINITY, L = 0.0f, y[HD / 2];
            for (uint32_t z = 0; z < parts; z++)
                M = fmaxf(M, __ldcg(part + (z * (HD + 2) + HD) * kRows));
#pragma unroll
            for (uint32_t k = 0; k < HD / 2; k++) y[k] = 0.0f;
            for (uint32_t z = 0; z < parts; z++) {
                const float* pz = part + z * ((HD + 2) * kRows);
                const float mz = __ldcg(pz + HD * kRows), lz = __ldcg(pz + (HD + 1) * kRows);
                const float f = mz == -INFINITY ? 0.0f : ex2(mz - M);
                L = fmaf(lz, f, L);
#pragma unroll
                for (uint32_t k = 0; k < HD / 2; k++)
                    y[k] = fmaf(__ldcg(pz + (half * (HD / 2) + k) * kRows), f, y[k]);
            }
            const float by = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
            for (uint32_t c = 0; c < HD / 32; c++) {
                float v[16];
#pragma unroll
                for (int k = 0; k < 16; k++) v[k] = y[16 * c + k] * by;
                if (live) put_out(p, orow, half * (HD / 2) + 16 * c, v);
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
    p.splits = (uint32_t)std::max<uint64_t>(1, s->rt->sm_count / units);
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
