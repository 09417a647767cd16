// attention.hip -- attention of a step's queries over a paged cache.
//
// out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, h / G]) v[j, h / G] over the keys j
// that token t sees: every cached key of its sequence and, of the call's new ones,
// those up to its own (a chain) or those whose bit is set in its mask (a tree).
#include <hip/hip_runtime.h>

#include "cache_device.h"

namespace mx4 {

// One workgroup a (token, head); 256 keys a pass, one a thread, with a running
// maximum m and sum l of exp(s - m).
template <int D>
__global__ __launch_bounds__(256) void attention_kernel(AttentionArgs a) {
    __shared__ float q[D], p[256], red[8], acc_part[256];
    const uint32_t t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t s = sequence_of(a.step.start, a.step.seqs, t);
    uint16_t* out = a.out + t * a.out_stride + (uint64_t)h * D;
    if (s >= a.step.seqs) return;
    uint32_t first, fresh;
    tokens_of(a.step, s, first, fresh);
    const uint32_t before = a.step.cached[s], i = t - first;
    if (i >= fresh) return;
    const uint32_t keys = min(before + fresh, table_room(a.step, a.cache.page_shift));
    const uint32_t kv = h / (a.q_heads / a.cache.kv_heads);
    for (uint32_t d = tid; d < D; d += 256)
        q[d] = __uint_as_float((uint32_t)a.q[t * a.q_stride + (uint64_t)h * D + d] << 16) * a.scale;
    const uint32_t* table = a.step.table + (uint64_t)s * a.step.table_stride;
    auto row = [&](uint32_t key) {
        const uint32_t page = min(table[key >> a.cache.page_shift], a.cache.pages - 1);
        return ((((uint64_t)page * a.cache.kv_heads + kv) << a.cache.page_shift) + (key & ((1u << a.cache.page_shift) - 1))) * D;
    };
    __syncthreads();
    constexpr int PARTS = 256 / (D < 256 ? D : 256);
    const uint32_t d = tid % D, part = tid / D;
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    for (uint32_t k0 = 0; k0 < keys; k0 += 256) {
        const uint32_t key = k0 + tid;
        bool sees = key < keys;
        if (sees && key >= before) {
            const uint32_t j = key - before;
            sees = a.tree ? j < 64 * a.tree_words && (a.tree[(uint64_t)t * a.tree_words + j / 64] >> (j % 64) & 1) : j <= i;
        }
        float dot = -INFINITY;
        if (sees) {
            dot = 0.0f;
            const uint16_t* k = a.cache.k + row(key);
            for (int e = 0; e < D; ++e) dot = __builtin_fmaf(q[e], __uint_as_float((uint32_t)k[e] << 16), dot);
        }
        float top = dot;
        for (int off = 1; off < 64; off *= 2) top = fmaxf(top, __shfl_xor(top, off));
        if (lane == 0) red[wave] = top;
        __syncthreads();
        const float now = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float base = now == -INFINITY ? 0.0f : now;
        const float weight = sees ? expf(dot - base) : 0.0f;
        p[tid] = sees ? weight : -1.0f;  // a key that is not seen is told from one that weighs nothing
        float sum = weight;
        for (int off = 1; off < 64; off *= 2) sum += __shfl_xor(sum, off);
        if (lane == 0) red[4 + wave] = sum;
        __syncthreads();
        const float keep = m == -INFINITY ? 0.0f : expf(m - base);
        m = now;
        l = l * keep + red[4] + red[5] + red[6] + red[7];
        acc *= keep;
        for (uint32_t e = part; e < 256 && k0 + e < keys; e += PARTS)
            if (!(p[e] < 0.0f)) acc = __builtin_fmaf(p[e], __uint_as_float((uint32_t)a.cache.v[row(k0 + e) + d] << 16), acc);
        __syncthreads();
    }
    acc_part[tid] = acc;
    __syncthreads();
    if (part == 0) {
        float sum = 0.0f;
        for (int e = 0; e < PARTS; ++e) sum += acc_part[e * D + d];
        const __bf16 o = (__bf16)(m == -INFINITY ? 0.0f : sum / l);
        out[d] = __builtin_bit_cast(uint16_t, o);
    }
}

hipError_t launch_attention(const AttentionArgs& a, int cus) {
    const dim3 grid(a.step.tokens, a.q_heads);
    if (a.cache.head_dim == 64) attention_kernel<64><<<grid, dim3(256), 0, a.stream>>>(a);
    if (a.cache.head_dim == 128) attention_kernel<128><<<grid, dim3(256), 0, a.stream>>>(a);
    if (a.cache.head_dim == 256) attention_kernel<256><<<grid, dim3(256), 0, a.stream>>>(a);
    return hipGetLastError();
}

}  // namespace mx4
