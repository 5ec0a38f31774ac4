// The 4-bit key/value cache: quantising rows as they are written, reading rows back, and the
// cache handle. Attention over it is in kv4_attention.cu.
//
// One vector is what one kv head keeps for one position: `head` values, held as 4-bit codes and
// one word with two bf16 numbers, the step s (low half) and the offset m (high half):
//     m = bf16(min x)   s = bf16(max(max x - m, 0) / 15)   c_i = rne((x_i - m) / s) in 0..15
// and standing for m + s c_i. A vector with a value that is not finite, or whose range is not,
// has NaN for both and reads back as NaN throughout. Element i is bits 4 (i % 8) and up of word
// i / 8; a row of codes is padded with zeros to a multiple of 16 bytes (32 elements). Arrays are
// head-major ([batch,] kv_heads, seq, words), so that the positions of one head are one
// contiguous run for the attention that streams them.
#include <algorithm>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "kv4.h"

namespace ab {

// ---- operands ---------------------------------------------------------------------------
Kv4View kv4_operands(const ab_kv4_layer& c, uint32_t rows, uint32_t kv_heads, uint32_t head) {
    static const char* names[4] = {"cache.key_codes", "cache.key_scales", "cache.value_codes",
                                   "cache.value_scales"};
    const ab_tensor t[4] = {c.key_codes, c.key_scales, c.value_codes, c.value_scales};
    for (int i = 0; i < 4; i++) {
        expect_data(names[i], t[i]);
        expect_dtype(names[i], t[i], AB_U32);
    }
    if (head == 0 || head > kKv4MaxHead)
        invalid("kv4: head size " + std::to_string(head) + " is not in 1..128");
    expect_rank_in(names[0], t[0], 3, 4);
    const int cr = t[0].rank;
    for (int i = 0; i < 4; i++) {
        expect_rank(names[i], t[i], i % 2 ? cr - 1 : cr);
        for (int a = 0; a < t[i].rank; a++)
            if (t[i].dims[a] != t[0].dims[a])
                invalid(std::string("parameter `") + names[i] +
                        "`: leading dims must match cache.key_codes " + shape_str(t[0]));
    }
    if (cr == 4 && t[0].dims[0] < rows) expect_dim(names[0], t[0], 0, "batch", rows);
    expect_dim(names[0], t[0], cr - 3, "kv_heads", kv_heads);
    expect_dim(names[0], t[0], cr - 1, "words", kv4_words(head));
    for (int i = 0; i < 4; i++)
        if ((uintptr_t)t[i].data % (i % 2 ? 4 : 16))
            invalid(std::string("parameter `") + names[i] + "`: must be " +
                    (i % 2 ? "4" : "16") + "-byte aligned");
    Kv4View v = {};
    v.kv_heads = kv_heads;
    v.head = head;
    v.seq = t[0].dims[cr - 2];
    v.words = t[0].dims[cr - 1];
    v.row_stride = cr == 4 ? (uint64_t)kv_heads * v.seq : 0;
    for (int w = 0; w < 2; w++) {
        v.codes[w] = (uint32_t*)t[2 * w].data;
        v.scales[w] = (uint32_t*)t[2 * w + 1].data;
    }
    return v;
}

namespace {

constexpr int kThreads = 256;
constexpr int kLoadUnroll = 4;  // vectors a lane group of the load has in flight

// 16 bytes that are read once. Not the non-coherent path: this grid may have started while the
// kernel that writes them still ran.
__device__ __forceinline__ uint4 ld_once(const void* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p));
    return r;
}

// Smaller and larger, NaN if either is.
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint32_t min_nan2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t max_nan2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Eight elements of a row as they were read: bf16 in pairs, f32.
template <typename T>
struct Eight;
template <>
struct Eight<float> {
    float v[8];
    __device__ __forceinline__ float at(int i) const { return v[i]; }
    __device__ __forceinline__ void load(const float* p) {
        const uint4 a = ld_once(p), b = ld_once(p + 4);
        v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y);
        v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
        v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y);
        v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
    }
    __device__ __forceinline__ void set(int i, float x) { v[i] = x; }
};
// Smallest and largest of a vector, two Eights (`any`: the first has elements; the second holds
// some of them) in each of LPV lanes; NaN if one is.
template <int LPV>
__device__ __forceinline__ void extremes(const Eight<float> (&e)[2], bool any, float* lo,
                                         float* hi) {
    float l = e[0].v[0], h = l;
#pragma unroll
    for (int i = 1; i < 16; i++) {
        l = min_nan(l, e[i / 8].v[i % 8]);
        h = max_nan(h, e[i / 8].v[i % 8]);
    }
    if (!any) {
        l = INFINITY;
        h = -INFINITY;
    }
#pragma unroll
    for (int o = LPV / 2; o > 0; o >>= 1) {
        l = min_nan(l, __shfl_xor_sync(0xffffffffu, l, o));
        h = max_nan(h, __shfl_xor_sync(0xffffffffu, h, o));
    }
    *lo = l;
    *hi = h;
}
template <>
struct Eight<bf16> {
    uint32_t w[4];
    __device__ __forceinline__ float at(int i) const {
        return i % 2 ? bf16hi(w[i / 2]) : bf16lo(w[i / 2]);
    }
    __device__ __forceinline__ void load(const bf16* p) {
        const uint4 a = ld_once(p);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    }
    __device__ __forceinline__ void set(int i, bf16 x) {
        const uint32_t b = __bfloat16_as_ushort(x);
        w[i / 2] = i % 2 ? w[i / 2] | b << 16 : b;
    }
};
// In pairs; then the smallest and minus the largest as one pair.
template <int LPV>
__device__ __forceinline__ void extremes(const Eight<bf16> (&e)[2], bool any, float* lo,
                                         float* hi) {
    uint32_t l = e[0].w[0], h = l;
#pragma unroll
    for (int i = 1; i < 8; i++) {
        l = min_nan2(l, e[i / 4].w[i % 4]);
        h = max_nan2(h, e[i / 4].w[i % 4]);
    }
    h ^= 0x80008000u;
    uint32_t x = min_nan2(__byte_perm(l, h, 0x5410), __byte_perm(l, h, 0x7632));
    if (!any) x = 0x7f807f80u;  // infinities
#pragma unroll
    for (int o = LPV / 2; o > 0; o >>= 1) x = min_nan2(x, __shfl_xor_sync(0xffffffffu, x, o));
    *lo = bf16lo(x);
    *hi = -bf16hi(x);
}
// `left` elements of the row exist from p on (vec: 16-byte loads, whole eights). Past the row's
// end its first element here stands again, which changes no extreme.
template <typename T>
__device__ __forceinline__ void load16(const T* p, uint32_t left, bool vec, Eight<T> (&e)[2]) {
    if (vec) {
        if (left) e[0].load(p);
        if (left > 8) e[1].load(p + 8);
        else e[1] = e[0];
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 16; i++)
            e[i / 8].set(i % 8, left ? p[i < left ? i : 0] : from_f32<T>(0.0f));
    }
}

// ---- codes -------------------------------------------------------------------------------
// The code of x is the whole number nearest to (x - m) / s in real arithmetic, halves to even,
// within 0..15. f = fl(fl(x - m) * fl(1 / (15 s))), cut to 0..1, times 15 is within 5 * 2^-24 * 15
// < 5e-6 of the quotient, which decides every case but those that close to a half.
//   f32 rows: these are about one word in ten thousand; exact_word decides them.
//   bf16 rows: quotients of 8-bit numbers, they are halves or well apart from them, and halves
//   are common. With k = rne(15 f) and d = x - m, d - k s is exact, and is +-s / 2 for a half: the
//   even neighbour is then 2 rne(7.5 f). d itself is inexact only where x is 2^16 below m, or m
//   below x: rows where the quotient next to that, -m / s or x / s, may be a half, go to
//   exact_word whole (m / s a half, one row in a hundred; 0 < |m| < s / 2^11).
constexpr float kNearHalf = 0.499995f;
constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number

// The same for a whole word, decided exactly in 32 bits. With d = fl(x - m) and its error e,
// x - m - h s has the sign of fma(-h, s, d) + e: h s (h a half, s of 8 bits) enters exactly, and
// where it is near d the difference is exact. Elements are read again: the caller's are in
// registers, and a loop keeps this path short.
template <typename T>
__device__ __noinline__ uint32_t exact_word(const T* p, uint32_t left, float m, float s) {
    const float up = s < 0x1p-100f ? 0x1p64f : 1.0f;  // a reciprocal that is a normal number
    const float inv = 1.0f / (s * up);
    uint32_t word = 0;
    for (uint32_t i = 0; i < min(left, 8u); i++) {
        const float x = to_f32(p[i]), d = x - m;
        const float back = d - x, e = (x - (d - back)) + (-m - back);
        float k = rintf(fminf(fmaxf(d * up * inv, 0.0f), 15.0f));
        const bool odd = ((int)k & 1) != 0;
        const float over = fmaf(-(k + 0.5f), s, d) + e, under = fmaf(0.5f - k, s, d) + e;
        if (over > 0.0f || (over == 0.0f && odd)) k += 1.0f;
        else if (under < 0.0f || (under == 0.0f && odd)) k -= 1.0f;
        word |= (uint32_t)fminf(fmaxf(k, 0.0f), 15.0f) << (4 * i);
    }
    return word;
}

constexpr uint32_t kRowsPerScan = 1024;

// ordered[i]: the rows [1024 i, 1024 (i + 1)] of the parcel are at strictly rising positions.
__global__ void __launch_bounds__(kRowsPerScan)
    kv4_order_kernel(const Step* step, uint32_t rows, uint32_t* ordered) {
    pdl_wait();
    pdl_trigger();
    const uint32_t r = blockIdx.x * kRowsPerScan + threadIdx.x;
    const bool ok = r + 1 >= rows || step[r].position < step[r + 1].position;
    const int all = __syncthreads_and(ok);
    if (threadIdx.x == 0) ordered[blockIdx.x] = all;
}

// LPV lanes hold one vector, sixteen elements (two code words) each; a block takes kThreads / LPV
// consecutive vectors of one of the two tensors (blockIdx.y), kv heads fastest, so its loads are
// one contiguous run of the source. Bound by instructions, 28 an element: 32768 bf16 rows of 8 x 128
// (170 MB) take 66 us, 2.6 TB/s with 82% of the issue slots used. With eight elements a lane, each
// vector's own work on twice the lanes, they took 88 us, with sixteen and four vectors a lane in
// flight 79: many blocks of an SM hide the loads better.
template <typename T, int LPV>
__global__ void __launch_bounds__(kThreads, 6)
    kv4_store_kernel(const T* key, const T* value, const Kv4View c,
                     uint32_t total, uint32_t rows, const Step* step, int vec,
                     const uint32_t* ordered, uint32_t* flags) {
    constexpr uint32_t VECS = kThreads / LPV;
    __shared__ uint32_t lost[VECS];  // per row of this block: a later row has its position
    pdl_wait();
    const uint32_t which = blockIdx.y;
    const T* src = which ? value : key;
    uint32_t* codes = which ? c.codes[1] : c.codes[0];
    uint32_t* scales = which ? c.scales[1] : c.scales[0];
    const uint32_t v0 = blockIdx.x * VECS;
    const uint32_t sub = threadIdx.x % LPV, grp = threadIdx.x / LPV;
    const uint32_t e0 = sub * 16;
    const uint32_t left = e0 < c.head ? c.head - e0 : 0;
    const uint32_t v = v0 + grp;
    const bool live = v < total;
    const uint32_t row = live ? v / c.kv_heads : 0, kvh = live ? v - row * c.kv_heads : 0;
    const T* mine = src + (live ? (uint64_t)v * c.head + e0 : 0);
    uint32_t pos = live ? step[row].position : 0xffffffffu;
    Eight<T> x[2];
    load16(mine, live ? left : 0, vec, x);
    if (live && pos >= c.seq && sub == 0) atomicOr(flags, kFlagPositionRange);
    // rows of one cache at the same position: the last one is written. Rising positions (a
    // prompt) cannot meet; otherwise the block looks through the rows after its own.
    bool scan = c.row_stride == 0 && rows > 1;
    if (scan && ordered) {
        bool ok = true;
        for (uint32_t i = threadIdx.x; i < (rows + kRowsPerScan - 1) / kRowsPerScan; i += kThreads)
            ok = ok && ordered[i] != 0;
        scan = !__syncthreads_and(ok);
    }
    if (scan) {
        const uint32_t r0 = v0 / c.kv_heads;
        const uint32_t r1 = min(rows, (v0 + VECS - 1) / c.kv_heads + 1);
        for (uint32_t r = threadIdx.x; r < VECS; r += kThreads) lost[r] = 0;
        __syncthreads();
        for (uint32_t q = r0 + 1 + threadIdx.x; q < rows; q += kThreads) {
            const uint32_t pq = step[q].position;
            for (uint32_t r = r0; r < min(q, r1); r++)
                if (step[r].position == pq) lost[r - r0] = 1;
        }
        __syncthreads();
        if (live && lost[row - r0]) pos = 0xffffffffu;
    }
    pdl_trigger();
    float lo, hi;
    extremes<LPV>(x, left != 0, &lo, &hi);
    const bf16 mb = __float2bfloat16_rn(lo);
    const float m = __bfloat162float(mb);
    const bf16 sb = __float2bfloat16_rn(__fdiv_rn(fmaxf(__fsub_rn(hi, m), 0.0f), 15.0f));
    const float s = __bfloat162float(sb);
    // a value of the row, its range or its offset is not finite
    const bool bad = !(isfinite(lo) && isfinite(hi) && isfinite(m) && isfinite(s));
    const bool write = pos < c.seq;
    uint32_t word[2] = {0, 0};
    if (!bad && s > 0.0f) {
        const float inv = 1.0f / (15.0f * s);
        // where 15 s or its reciprocal leaves the normal numbers
        bool exactly = s < 0x1p-100f || s > 0x1p120f;
        if constexpr (sizeof(T) == 2) {
            const float q = -m * inv, twice = fmaf(q, 30.0f, kMagic) - kMagic;
            exactly |= (q > 0.0f && q < 1.1f && fmaf(0.5f * twice, s, m) == 0.0f &&
                        ((int)twice & 1)) ||
                       (m != 0.0f && fabsf(m) < s * 0x1p-11f);
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
            float near = 0.0f;
            // eight codes, each with kMagic's bits above it, as digits of base 16
#pragma unroll
            for (int i = 7; i >= 0; i--) {
                const float d = x[j].at(i) - m, f = __saturatef(d * inv);
                float k = fmaf(f, 15.0f, kMagic);
                if constexpr (sizeof(T) == 4) {
                    near = fmaxf(near, fabsf(fmaf(f, 15.0f, kMagic - k)));
                } else {
                    const float even = fmaf(f, 7.5f, kMagic) - kMagic;
                    if (fabsf(fmaf(kMagic - k, s, d)) == 0.5f * s) k = fmaf(even, 2.0f, kMagic);
                }
                word[j] = word[j] * 16 + __float_as_uint(k);
            }
            word[j] -= 0x4b400000u * 0x11111111u;
            const uint32_t here = left > 8u * j ? left - 8 * j : 0;
            if ((exactly || near > kNearHalf) && write)
                word[j] = exact_word(mine + 8 * j, here, m, s);
            if (here < 8) word[j] &= here ? 0xffffffffu >> (32 - 4 * here) : 0u;
        }
    }
    if (!write) return;
    const uint64_t at = (uint64_t)row * c.row_stride + (uint64_t)kvh * c.seq + pos;
    if (2 * sub < c.words)
        *reinterpret_cast<uint2*>(codes + at * c.words + 2 * sub) = make_uint2(word[0], word[1]);
    if (sub == 0)
        scales[at] = bad ? 0x7fff7fffu
                         : (uint32_t)__bfloat16_as_ushort(sb) |
                               ((uint32_t)__bfloat16_as_ushort(mb) << 16);
}

// ---- values ------------------------------------------------------------------------------
// The eight values of a code word, in order, rounded once to the output's type. A code becomes a
// number by standing in the low bits of one whose units these are (bf16 128, f32 2^23), which is
// then taken off; bf16 goes two at a time, elements i and i + 4 of the word.
__device__ __forceinline__ void values_of(uint32_t word, uint32_t sc, uint32_t (&v)[4]) {
    const uint32_t s2 = __byte_perm(sc, sc, 0x1010), m2 = __byte_perm(sc, sc, 0x3232);
    uint32_t p[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t x = (word >> (4 * j) & 0x000f000fu) | 0x43004300u;
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(p[j]) : "r"(x), "r"(0x43004300u));
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(p[j]) : "r"(p[j]), "r"(s2), "r"(m2));
    }
    v[0] = __byte_perm(p[0], p[1], 0x5410);
    v[1] = __byte_perm(p[2], p[3], 0x5410);
    v[2] = __byte_perm(p[0], p[1], 0x7632);
    v[3] = __byte_perm(p[2], p[3], 0x7632);
}
__device__ __forceinline__ void values_of(uint32_t word, uint32_t sc, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float x = __uint_as_float((word >> (4 * i) & 15u) | 0x4b000000u);
        v[i] = fmaf(x - 8388608.0f, bf16lo(sc), bf16hi(sc));
    }
}
// 16 bytes of values, or those of them that the row has (`left`).
__device__ __forceinline__ void put16(bf16* p, const uint32_t (&v)[4], uint32_t left, bool vec) {
    if (vec) {
        *reinterpret_cast<uint4*>(p) = make_uint4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; i++)
            if (i < left) p[i] = __ushort_as_bfloat16((unsigned short)(v[i / 2] >> (16 * (i % 2))));
    }
}
__device__ __forceinline__ void put16(float* p, const float (&v)[4], uint32_t left, bool vec) {
    if (vec) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
            if (i < left) p[i] = v[i];
    }
}

// Vectors go to lane groups in order, kv heads fastest: a group's next one is GROUPS further,
// `lines` positions and `heads` heads on.
struct Walk {
    uint32_t total, lines, heads;
};

// Reading back: LPV lanes a vector, 16 bytes of output each (eight bf16 values, a code word, or
// four f32 values, half of one), so that a warp's stores are whole lines: with eight f32 values a
// lane, 16 streams of 1000 positions of 12 x 64 took 30 us, so 25 (112 MB, 4.5 TB/s). As bf16,
// 131072 positions of 8 x 128 take 110 us: 680 MB at 6.1 TB/s, 0.94 of a copy's rate. Output row i
// of batch row b is position step[b].position + i; positions past the cache's end give zeros and
// raise the position flag.
template <typename T, int LPV>
__global__ void __launch_bounds__(kThreads)
    kv4_load_kernel(T* key, T* value, const Kv4View c, const Walk walk, uint32_t n,
                    const Step* step, int vec, uint32_t* flags) {
    constexpr uint32_t GROUPS = kThreads / LPV;
    constexpr uint32_t PER = 16 / sizeof(T);  // values of a lane
    pdl_wait();
    pdl_trigger();
    const uint32_t which = blockIdx.y;
    T* dst = which ? value : key;
    const uint32_t* codes = which ? c.codes[1] : c.codes[0];
    const uint32_t* scales = which ? c.scales[1] : c.scales[0];
    const uint32_t sub = threadIdx.x % LPV, grp = threadIdx.x / LPV;
    const uint32_t e0 = sub * PER;
    const uint32_t v0 = blockIdx.x * (GROUPS * kLoadUnroll) + grp;
    uint32_t line = v0 / c.kv_heads, kvh = v0 - line * c.kv_heads;
    uint32_t b = line / n, i = line - b * n;
    uint32_t word[kLoadUnroll], sc[kLoadUnroll];
#pragma unroll
    for (int u = 0; u < kLoadUnroll; u++) {
        word[u] = sc[u] = 0;
        if (v0 + u * GROUPS < walk.total) {
            const uint64_t pos = (uint64_t)step[b].position + i;
            if (pos < c.seq) {
                const uint64_t at = (uint64_t)b * c.row_stride + (uint64_t)kvh * c.seq + pos;
                if (e0 < 8 * c.words) word[u] = __ldcg(codes + at * c.words + e0 / 8) >> 4 * (e0 % 8);
                sc[u] = __ldcg(scales + at);
            } else if (sub == 0) {
                atomicOr(flags, kFlagPositionRange);
            }
        }
        kvh += walk.heads;
        i += walk.lines;
        if (kvh >= c.kv_heads) {
            kvh -= c.kv_heads;
            i++;
        }
        if (i >= n) {
            b += i / n;
            i %= n;
        }
    }
#pragma unroll
    for (int u = 0; u < kLoadUnroll; u++) {
        const uint32_t v = v0 + u * GROUPS;
        if (v >= walk.total || e0 >= c.head) continue;
        typename std::conditional<sizeof(T) == 2, uint32_t[4], float[4]>::type x;
        values_of(word[u], sc[u], x);
        put16(dst + (uint64_t)v * c.head + e0, x, c.head - e0, vec);
    }
}

// Rows [n, kv_heads, head], or [kv_heads, head] for one; both tensors alike.
struct Kv4Rows {
    uint32_t rows, kv_heads, head, vectors;
    int vec;  // 16-byte accesses: whole groups of eight elements, aligned
};

Kv4Rows rows_of(const ab_tensor& key, const ab_tensor& value, int rank_lo, int rank_hi) {
    expect_data("key", key);
    expect_data("value", value);
    expect_float("key", key);
    expect_dtype("value", value, key.dtype);
    expect_rank_in("key", key, rank_lo, rank_hi);
    expect_rank("value", value, key.rank);
    for (int a = 0; a < key.rank; a++)
        if (value.dims[a] != key.dims[a])
            invalid("parameter `value`: dims must match key " + shape_str(key));
    Kv4Rows r = {};
    r.head = key.dims[key.rank - 1];
    r.kv_heads = key.dims[key.rank - 2];
    const uint64_t rows = numel(key) / ((uint64_t)r.head * r.kv_heads);
    if ((rows * r.kv_heads) >> 31) invalid("parameter `key`: too many vectors for one call");
    if (((uintptr_t)key.data | (uintptr_t)value.data) % dtype_size(key.dtype))
        invalid("parameter `key` / `value`: not aligned to its elements");
    r.rows = (uint32_t)rows;
    r.vectors = r.rows * r.kv_heads;
    r.vec = r.head % 8 == 0 && ((uintptr_t)key.data | (uintptr_t)value.data) % 16 == 0;
    return r;
}

// Calls f with the power of two of lanes that covers a vector.
template <typename F>
void with_lanes(uint32_t lanes, F&& f) {
    if (lanes <= 2) f(std::integral_constant<int, 2>());
    else if (lanes <= 4) f(std::integral_constant<int, 4>());
    else if (lanes <= 8) f(std::integral_constant<int, 8>());
    else if (lanes <= 16) f(std::integral_constant<int, 16>());
    else f(std::integral_constant<int, 32>());
}

unsigned blocks_for(uint32_t vectors, uint32_t per_block) {
    return (unsigned)(((uint64_t)vectors + per_block - 1) / per_block);
}

}  // namespace

void record_kv4_store(ab_scheme* s, const char* label, ab_tensor key, ab_tensor value,
                      const ab_kv4_layer& cache, ab_tensor step) {
    const Kv4Rows r = rows_of(key, value, 2, 3);
    const Kv4View c = kv4_operands(cache, r.rows, r.kv_heads, r.head);
    expect_step(step, r.rows);
    const Step* st = (const Step*)step.data;
    uint32_t* flags = s->rt ? s->rt->flags : nullptr;
    // Rows over one cache: every block looks for later rows at its rows' positions. Where that
    // takes a thread more than 512 comparisons (about 1 us), whether the positions rise is
    // settled once instead, by a kernel of its own.
    uint32_t* ordered = nullptr;
    const uint32_t chunks = (r.rows + kRowsPerScan - 1) / kRowsPerScan;
    const uint64_t block_rows = kThreads / std::max(2u, c.words / 2) / r.kv_heads + 2;
    if (c.row_stride == 0 && r.rows / kThreads * block_rows > 512 && s->rt) {
        s->rt->activate();
        cuda_check(cudaMalloc((void**)&ordered, chunks * 4ull), "cudaMalloc");
        s->owned.push_back(ordered);
        s->add("kv4_order", [=](cudaStream_t stream) {
            return launch(stream, dim3(chunks), dim3(kRowsPerScan), 0, true, kv4_order_kernel, st,
                          r.rows, ordered);
        });
    }
    with_lanes(c.words / 2, [&](auto lanes) {
        constexpr int LPV = decltype(lanes)::value;
        if constexpr (LPV <= 8) {  // 16 words at most
            const unsigned blocks = blocks_for(r.vectors, kThreads / LPV);
            auto go = [&](auto tag) {
                using T = decltype(tag);
                const T *k = (const T*)key.data, *v = (const T*)value.data;
                s->add(label, [=](cudaStream_t stream) {
                    return launch(stream, dim3(blocks, 2), dim3(kThreads), 0, true,
                                  kv4_store_kernel<T, LPV>, k, v, c, r.vectors, r.rows, st, r.vec,
                                  (const uint32_t*)ordered, flags);
                });
            };
            if (key.dtype == AB_F32) go(float());
            else go(bf16());
        }
    });
}

}  // namespace ab

using namespace ab;

struct ab_kv4cache {
    Runtime* rt;
    uint32_t layers, batch, seq, kv_heads, head;
    void* data[4];  // key codes, key scales, value codes, value scales
    uint64_t vectors() const { return (uint64_t)layers * batch * kv_heads * seq; }
    uint64_t bytes(int i) const { return vectors() * (i % 2 ? 4 : 4ull * kv4_words(head)); }
};

extern "C" {

int ab_kernel_kv4_store(ab_scheme* s, ab_tensor key, ab_tensor value, const ab_kv4_layer* cache,
                        ab_tensor step) {
    return guard([&] {
        if (!s || !cache) fail(AB_ERR_ARGUMENT, "null argument");
        record_kv4_store(s, "kv4_store", key, value, *cache, step);
    });
}

int ab_kernel_kv4_load(ab_scheme* s, const ab_kv4_layer* cache, ab_tensor step, ab_tensor key,
                       ab_tensor value) {
    return guard([&] {
        if (!s || !cache) fail(AB_ERR_ARGUMENT, "null argument");
        const Kv4Rows r = rows_of(key, value, 3, 4);
        const uint32_t batch = key.rank == 4 ? key.dims[0] : 1;
        const uint32_t n = key.dims[key.rank - 3];
        const Kv4View c = kv4_operands(*cache, batch, r.kv_heads, r.head);
        if (n > c.seq) invalid("parameter `key`: " + std::to_string(n) +
                               " positions from a cache of " + std::to_string(c.seq));
        expect_step(step, batch);
        const Step* st = (const Step*)step.data;
        uint32_t* flags = s->rt ? s->rt->flags : nullptr;
        auto go = [&](auto tag) {
            using T = decltype(tag);
            T *k = (T*)key.data, *v = (T*)value.data;
            with_lanes(c.words * sizeof(T) / 2, [&](auto lanes) {
                constexpr int LPV = decltype(lanes)::value;
                constexpr uint32_t GROUPS = kThreads / LPV;
                const unsigned blocks = blocks_for(r.vectors, GROUPS * kLoadUnroll);
                const Walk walk{r.vectors, GROUPS / r.kv_heads, GROUPS % r.kv_heads};
                s->add("kv4_load", [=](cudaStream_t stream) {
                    return launch(stream, dim3(blocks, 2), dim3(kThreads), 0, true,
                                  kv4_load_kernel<T, LPV>, k, v, c, walk, n, st, r.vec, flags);
                });
            });
        };
        if (key.dtype == AB_F32) go(float());
        else go(bf16());
    });
}

int ab_kv4cache_create(ab_runtime* rt, uint32_t layers, uint32_t seq_len, uint32_t kv_heads,
                       uint32_t head_size, uint32_t batch, ab_kv4cache** out) {
    return guard([&] {
        if (!rt || !out) fail(AB_ERR_ARGUMENT, "null argument");
        if (!layers || !seq_len || !kv_heads || !head_size || !batch)
            fail(AB_ERR_ARGUMENT, "Kv4Cache dims must be non-zero");
        if (head_size > kKv4MaxHead)
            fail(AB_ERR_ARGUMENT, "Kv4Cache head size must be at most 128");
        if ((double)layers * seq_len * kv_heads * batch > (double)(1ull << 40))
            fail(AB_ERR_ARGUMENT, "Kv4Cache dims must make at most 2^40 vectors");
        auto* c = new ab_kv4cache{rt, layers, batch, seq_len, kv_heads, head_size, {}};
        try {
            rt->activate();
            for (int i = 0; i < 4; i++) {
                cuda_check(cudaMalloc(&c->data[i], c->bytes(i)), "cudaMalloc");
                cuda_check(clear_device(rt, c->data[i], c->bytes(i)), "clear");
            }
        } catch (...) {
            for (void* p : c->data)
                if (p) cudaFree(p);
            delete c;
            throw;
        }
        *out = c;
    });
}

int ab_kv4cache_layer(const ab_kv4cache* c, uint32_t layer, ab_kv4_layer* out) {
    return guard([&] {
        if (!c || !out) fail(AB_ERR_ARGUMENT, "null argument");
        if (layer >= c->layers)
            invalid("Kv4Cache::layer: layer " + std::to_string(layer) + " out of range (" +
                    std::to_string(c->layers) + " layers)");
        ab_tensor* t[4] = {&out->key_codes, &out->key_scales, &out->value_codes,
                           &out->value_scales};
        for (int i = 0; i < 4; i++) {
            *t[i] = ab_tensor{};
            t[i]->data = (char*)c->data[i] + layer * (c->bytes(i) / c->layers);
            t[i]->dtype = AB_U32;
            if (c->batch > 1) t[i]->dims[t[i]->rank++] = c->batch;
            t[i]->dims[t[i]->rank++] = c->kv_heads;
            t[i]->dims[t[i]->rank++] = c->seq;
            if (i % 2 == 0) t[i]->dims[t[i]->rank++] = kv4_words(c->head);
        }
    });
}

int ab_kv4cache_zero(ab_kv4cache* c) {
    return guard([&] {
        if (!c) fail(AB_ERR_ARGUMENT, "null cache");
        c->rt->activate();
        for (int i = 0; i < 4; i++)
            cuda_check(cudaMemsetAsync(c->data[i], 0, c->bytes(i), c->rt->stream), "zero cache");
    });
}

int ab_kv4cache_destroy(ab_kv4cache* c) {
    return guard([&] {
        if (!c) return;
        c->rt->activate();
        cudaStreamSynchronize(c->rt->stream);
        for (void* p : c->data) cudaFree(p);
        delete c;
    });
}

}  // extern "C"
