// The 4-bit key/value cache as the kernels see it (kv4.cu, kv4_attention.cu).
#pragma once

#include "internal.h"

namespace ab {

struct Step;

constexpr uint32_t kKv4MaxHead = 128;

// 32-bit words of one vector's codes: eight elements a word, rows padded to 16 bytes.
__host__ __device__ inline uint32_t kv4_words(uint32_t head) { return 4 * ((head + 31) / 32); }

// One layer: codes [B,] kv_heads, seq, words and scales [B,] kv_heads, seq for keys (0) and
// values (1). row_stride: vectors between the caches of consecutive rows (0: rows share one).
struct Kv4View {
    uint32_t* codes[2];
    uint32_t* scales[2];
    uint64_t row_stride;
    uint32_t kv_heads, seq, head, words;
};

// Checks a layer for `rows` rows of kv_heads heads of size head.
Kv4View kv4_operands(const ab_kv4_layer& c, uint32_t rows, uint32_t kv_heads, uint32_t head);

// Quantises rows key/value [rows, kv_heads, head] into the cache at step[row].position.
void record_kv4_store(ab_scheme* s, const char* label, ab_tensor key, ab_tensor value,
                      const ab_kv4_layer& cache, ab_tensor step);
// Attention of q [rows, heads, head] over a checked layer's positions 0 .. step[row].position.
void record_kv4_attention(ab_scheme* s, const char* label, const float* q, uint32_t rows,
                          uint32_t heads, const Kv4View& cache, void* out, int32_t out_dtype,
                          const Step* step);
// The same for rows of one shared cache and bf16 outputs on tcgen05 (kv4_prompt_tc.cu); false
// when the call is not one it takes.
bool record_kv4_prompt_tc(ab_scheme* s, const char* label, const float* q, uint32_t rows,
                          uint32_t heads, const Kv4View& cache, void* out, const Step* step);
// The scheme's scratch for parts and tickets (zero between launches). Its nodes run one after
// the other, so they share it; a node that needs more makes it anew for itself and later ones.
void kv4_take_scratch(ab_scheme* s, uint64_t part_bytes, uint64_t tickets, float** part,
                      uint32_t** ticket);

#ifdef __CUDACC__
// One arrival at a ticket: what the block wrote before its last barrier is published with it,
// what the earlier arrivals published is seen after it.
__device__ __forceinline__ uint32_t kv4_arrive(uint32_t* ticket) {
    uint32_t before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                 : "=r"(before)
                 : "l"(ticket)
                 : "memory");
    return before;
}
#endif

}  // namespace ab
