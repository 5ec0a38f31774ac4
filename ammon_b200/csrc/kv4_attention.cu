// Attention over the 4-bit key/value cache (format: kv4.cu).
//
// With k'_t = m_t + s_t c_t for the key at position t (and v'_t alike for the value),
//     score_t = (q . k'_t) / sqrt(head) = (s_t (q . c_t) + m_t sum q) / sqrt(head)
//     out = sum_t p_t (s_t c_t + m_t),  p = softmax over positions 0 .. the row's own.
// Scores, the softmax's maximum and sum and the output sums are held in 32 bits.
#include <algorithm>
#include <string>

#include "common.cuh"
#include "internal.h"
#include "kv4.h"

namespace ab {

namespace {

struct Kv4AttnParams {
    const float* q;  // [rows, heads, head]
    void* out;       // [rows, heads * head]
    Kv4View c;
    uint32_t rows, heads, group;
    const Step* step;
    uint32_t* flags;
};

constexpr int kWarps = 4;

// One block per (query head, row); its warps take every fourth position, a lane four elements.
template <typename OT>
__global__ void __launch_bounds__(kWarps * 32) kv4_attention_kernel(const Kv4AttnParams p) {
    __shared__ float sm[kWarps], sl[kWarps], so[kWarps][kKv4MaxHead];
    pdl_wait();
    pdl_trigger();
    const uint32_t h = blockIdx.x, r = blockIdx.y, hd = p.c.head;
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const uint32_t pos = p.step[r].position;
    if (pos >= p.c.seq && h == 0 && threadIdx.x == 0) atomicOr(p.flags, kFlagPositionRange);
    const uint32_t n = pos < p.c.seq ? pos + 1 : 0;
    const float* qr = p.q + ((uint64_t)r * p.heads + h) * hd;
    const float rs = 1.0f / sqrtf((float)hd);
    // sums of 256 positions are added to sums of these: a long run loses no digits to its length
    float q[4], qsum = 0.0f, acc[4] = {}, far[4] = {}, m = -INFINITY, l = 0.0f, lfar = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        q[i] = lane * 4 + i < hd ? qr[lane * 4 + i] * rs : 0.0f;
        qsum += q[i];
    }
    qsum = warp_sum(qsum);
    const uint64_t base = (uint64_t)r * p.c.row_stride + (uint64_t)(h / p.group) * p.c.seq;
    const uint32_t halves = p.c.words * 2;
    for (uint32_t t = warp; t < n; t += kWarps) {
        const uint16_t* kc = (const uint16_t*)p.c.codes[0] + (base + t) * halves;
        const uint16_t* vc = (const uint16_t*)p.c.codes[1] + (base + t) * halves;
        const uint32_t kw = lane < halves ? kc[lane] : 0, vw = lane < halves ? vc[lane] : 0;
        const uint32_t ks = p.c.scales[0][base + t], vs = p.c.scales[1][base + t];
        float d = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) d = fmaf(q[i], (float)((kw >> (4 * i)) & 15u), d);
        const float s = fmaf(bf16lo(ks), warp_sum(d), bf16hi(ks) * qsum);
        const float mn = fmaxf(m, s), a = expf(m - mn), e = expf(s - mn);
        m = mn;
        l = fmaf(l, a, e);
        lfar *= a;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            acc[i] = fmaf(acc[i], a,
                          e * fmaf((float)((vw >> (4 * i)) & 15u), bf16lo(vs), bf16hi(vs)));
            far[i] *= a;
        }
        if (t / kWarps % 256 == 255) {
            lfar += l;
            l = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                far[i] += acc[i];
                acc[i] = 0.0f;
            }
        }
    }
    l += lfar;
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] += far[i];
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) so[warp][lane * 4 + i] = acc[i];
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < hd; e += kWarps * 32) {
        float M = -INFINITY, L = 0.0f, o = 0.0f;
        for (int w = 0; w < kWarps; w++) M = fmaxf(M, sm[w]);
        for (int w = 0; w < kWarps; w++) {
            // a warp without positions has nothing; a NaN score must reach the output
            const float a = sm[w] == -INFINITY && sl[w] == 0.0f ? 0.0f : expf(sm[w] - M);
            L = fmaf(sl[w], a, L);
            o = fmaf(so[w][e], a, o);
        }
        ((OT*)p.out)[((uint64_t)r * p.heads + h) * hd + e] = from_f32<OT>(n ? o / L : 0.0f);
    }
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
        if (rows > 65535) invalid("parameter `q`: more than 65535 rows");
        p.q = (const float*)q.data;
        p.out = out.data;
        p.rows = rows;
        p.heads = heads;
        p.group = heads / kv;
        p.step = (const Step*)step.data;
        p.flags = s->rt ? s->rt->flags : nullptr;
        const bool f32 = out.dtype == AB_F32;
        s->add("kv4_attention", [=](cudaStream_t stream) {
            return launch(stream, dim3(heads, rows), dim3(kWarps * 32), 0, true,
                          f32 ? kv4_attention_kernel<float> : kv4_attention_kernel<bf16>, p);
        });
    });
}
