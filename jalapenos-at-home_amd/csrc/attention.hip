// attention.hip -- attention of a step's queries over a paged cache.
//
// out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, h / G]) v[j, h / G] over the keys j
// that token t sees: every cached key of its sequence and, of the call's new ones,
// those up to its own (a chain) or those whose bit is set in its mask (a tree).
//
// One pass over the keys with a running maximum m and sum l (of the weights as the
// matrix cores see them): p = 2^(s c - m), c = scale log2(e). A row's new tokens'
// query heads of one kv head share its keys, so they are the rows of one product:
// row r of a sequence is head h G + r % G of its new token r / G.
#include <hip/hip_runtime.h>

#include "attention_device.h"

namespace mx4 {

namespace {

// ------------------------------------------------------------- few rows a sequence

// A workgroup's four waves take the chunk's steps of 32 keys in turn, each with all
// 16 NT rows, keys and values straight from memory to registers. S^T = K Q^T
// leaves lane (row n = lane % 16, group g = lane / 16) the scores of keys 4 g .. 4 g + 3
// of each half step, which is what the next product's operand P^T wants from it if the
// values come in the same order -- so weights never cross lanes. A lane loads the 8 keys
// of its group at 8 neighbouring channels, and the 8 x 8 block turned round in
// registers (one v_perm a word) serves as the operand V^T of 8 products, channel
// 8 (lane % 16) + m in the m-th.
template <int D, int NT>
__global__ __launch_bounds__(256, NT <= 2 && D <= 128 ? 2 : 1) void attention_rows_kernel(AttentionArgs a, Split split,
                                                                                          uint32_t slot_rows) {
    constexpr int KK = D / 32, MT = D / 16, ROWS = 16 * NT, PITCH = D + 4;
    constexpr int CH = D >= 128 ? 8 : D / 16, VL = D / 16 / CH;  // channels of a value load, loads a key
    __shared__ float sums[4][16][PITCH];
    __shared__ float tops[4][ROWS];
    __shared__ float lsum[4][16];
    const uint32_t tid = threadIdx.x, lane = tid & 63, n16 = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t kv = blockIdx.y, group = a.q_heads / a.cache.kv_heads, shift = a.cache.page_shift;
    const uint32_t room = table_room(a.step, shift);
    Chunk c;
    if (!find_chunk(a.step, room, group, split, blockIdx.x, false, c)) return;
    const uint32_t seq = __builtin_amdgcn_readfirstlane(c.s);
    const Lengths n = lengths_of(a.step, seq, room);
    const uint32_t row0 = c.block * ROWS, rows = n.fresh * group - row0;  // rows of this block: min(rows, ROWS)

    // the queries, as the second operand of S^T
    bf16x8 q[NT][KK];
    uint32_t token[NT];  // new token of the lane's row, past the end: no row
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const uint32_t r = row0 + t * 16 + n16;
        token[t] = t * 16 + n16 < rows ? r / group : 0xffffffffu;
        const uint16_t* from = a.q + (uint64_t)(n.first + r / group) * a.q_stride + (uint64_t)(kv * group + r % group) * D + g * 8;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            u32x4 w = {0, 0, 0, 0};
            if (token[t] != 0xffffffffu) w = *reinterpret_cast<const u32x4*>(from + kk * 32);
            q[t][kk] = __builtin_bit_cast(bf16x8, w);
        }
    }
    const float cs = a.scale * 1.44269504088896340736f;

    const uint32_t step0 = c.chunk * c.cu * (kUnit / 32);
    const uint32_t step_end = min(step0 + c.cu * (kUnit / 32), (n.keys + 31) / 32);
    const uint32_t* table = a.step.table + (uint64_t)seq * a.step.table_stride;
    const uint32_t in_page = (1u << shift) - 1;

    f32x4 acc[NT][MT], lacc[NT];
    float top[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        top[t] = kNoMax;
        lacc[t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[t][m] = f32x4{0, 0, 0, 0};
    }
    bf16x8 ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = (__bf16)1.0f;

    u32x4 kf[2][KK];
    uint32_t vf[8][D / 32];  // 8 keys, the lane's D / 16 channels in pairs
    uint32_t pages = 0;      // lane 2 i + half: the page of this wave's i-th step from pages_at on
    auto load_pages = [&](uint32_t step) {
        const uint32_t key = (step + (lane >> 1) * 4) * 32 + (lane & 1) * 16;
        pages = min(table[min(key >> shift, a.step.table_stride - 1)], a.cache.pages - 1);
    };
    auto load = [&](uint32_t step, uint32_t i, u32x4 (&kd)[2][KK], uint32_t (&vd)[8][D / 32]) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t page = __builtin_amdgcn_readlane(pages, 2 * i + half);
            const uint64_t at = ((((uint64_t)page * a.cache.kv_heads + kv) << shift) + ((step * 32 + half * 16) & in_page)) * D;
            const uint16_t* kp = a.cache.k + at;
            const uint16_t* vp = a.cache.v + at;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) kd[half][kk] = *reinterpret_cast<const u32x4*>(kp + n16 * D + kk * 32 + g * 8);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < VL; ++e) {
                    const uint16_t* from = vp + (g * 4 + j) * D + e * 128 + n16 * CH;
                    if (CH == 8) {
                        const u32x4 w = *reinterpret_cast<const u32x4*>(from);
#pragma unroll
                        for (int x = 0; x < 4; ++x) vd[half * 4 + j][e * 4 + x] = w[x];
                    } else {
                        const uint2 w = *reinterpret_cast<const uint2*>(from);
                        vd[half * 4 + j][0] = w.x;
                        vd[half * 4 + j][1] = w.y;
                    }
                }
        }
    };

    uint32_t step = step0 + wave, i = 0;
    if (step < step_end) {
        load_pages(step);
        load(step, 0, kf, vf);
    }
    while (step < step_end) {
        u32x4 kn[2][KK];
        uint32_t vn[8][D / 32];
        const uint32_t next = step + 4;
        if (next < step_end) {
            if (++i == 32) {
                load_pages(next);
                i = 0;
            }
            load(next, i, kn, vn);
        }
        const uint32_t k0 = step * 32;
        const bool whole = k0 + 32 <= n.before;  // every row sees every key
        uint32_t bad = 0;
        if (!whole) {
            // values of keys that are not there count as zeros; of new tokens' values those
            // that are not finite are taken out here and added below for the rows that see them
            bool found = false;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool there = k0 + (j / 4) * 16 + g * 4 + j % 4 < n.keys;
#pragma unroll
                for (int x = 0; x < D / 32; ++x) {
                    if (!there) vf[j][x] = 0;
                    if (not_finite(vf[j][x])) {
                        found = true;
                        vf[j][x] = finite_only(vf[j][x]);
                    }
                }
            }
            bad = __any(found);
        }
        // V^T operands: words (key 2 e, key 2 e + 1) of channel m
        bf16x8 vt[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = __builtin_amdgcn_perm(vf[2 * e + 1][m / 2], vf[2 * e][m / 2], m % 2 ? 0x07060302u : 0x05040100u);
            vt[m] = __builtin_bit_cast(bf16x8, w);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            f32x4 s[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    s[half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kf[half][kk]), q[t][kk], s[half], 0, 0, 0);
            uint32_t seen = ~0u;
            if (!whole) {
                seen = token[t] != 0xffffffffu ? seen_window(a, n, token[t], k0) : 0u;
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(seen >> (half * 16 + g * 4 + e) & 1)) s[half][e] = -INFINITY;
            }
            float most = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                               fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3]))) * cs;
            if (__any(most > top[t] + kSlack)) {
                most = fmaxf(most, __shfl_xor(most, 16));
                most = fmaxf(most, __shfl_xor(most, 32));
                const float now = fmaxf(top[t], most), keep = __builtin_amdgcn_exp2f(top[t] - now);
                top[t] = now;
                lacc[t] *= keep;
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[t][m] *= keep;
            }
            bf16x8 p;  // rounded to bf16 for the product; the sum below takes the rounded ones
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = (__bf16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[e / 4][e % 4], cs, -top[t]));
            lacc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p, lacc[t], 0, 0, 0);
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[t][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt[m], p, acc[t][m], 0, 0, 0);
            if (bad) {
                // key by key: its weight in each row, its values again from memory
                for (uint32_t key = 0; key < 32 && k0 + key < n.keys; ++key) {
                    const uint32_t e = key / 16 * 4 + key % 4, page = min(table[(k0 + key) >> shift], a.cache.pages - 1);
                    float w = 0.0f;
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        if ((uint32_t)x == e) w = (float)p[x];
                    w = __shfl(w, key % 16 / 4 * 16 + n16);
                    const uint16_t* vp = a.cache.v + ((((uint64_t)page * a.cache.kv_heads + kv) << shift) + ((k0 + key) & in_page)) * D;
                    if (!(seen >> key & 1)) w = 0.0f;
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const uint32_t bits = vp[m / CH * 128 + (g * 4 + x) * CH + m % CH];
                            if ((bits & 0x7f80u) == 0x7f80u && (seen >> key & 1)) acc[t][m][x] += w * __uint_as_float(bits << 16);
                        }
                }
            }
        }
        step = next;
        if (next < step_end) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) kf[half][kk] = kn[half][kk];
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int x = 0; x < D / 32; ++x) vf[j][x] = vn[j][x];
        }
    }

    // the four waves' rows against one maximum, then their sum
    if (g == 0) {
#pragma unroll
        for (int t = 0; t < NT; ++t) tops[wave][t * 16 + n16] = top[t];
    }
    __syncthreads();
    float* part = a.part + ((uint64_t)(c.slot + c.chunk) * gridDim.y + kv) * slot_rows * (D + 2);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const uint32_t at = t * 16 + n16;
        const float now = fmaxf(fmaxf(tops[0][at], tops[1][at]), fmaxf(tops[2][at], tops[3][at]));
        const float keep = __builtin_amdgcn_exp2f(top[t] - now);
        if (t) __syncthreads();
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int m = 0; m < MT; ++m) sums[wave][n16][m / CH * 128 + (g * 4 + x) * CH + m % CH] = acc[t][m][x] * keep;
        if (g == 0) lsum[wave][n16] = lacc[t][0] * keep;
        __syncthreads();
        const uint32_t r = tid / 16, row = t * 16 + r, d0 = tid % 16 * (D / 16);
        if (row < rows) {
            const float l = (lsum[0][r] + lsum[1][r]) + (lsum[2][r] + lsum[3][r]);
            float o[D / 16];
#pragma unroll
            for (int x = 0; x < D / 16; ++x)
                o[x] = (sums[0][r][d0 + x] + sums[1][r][d0 + x]) + (sums[2][r][d0 + x] + sums[3][r][d0 + x]);
            if (c.chunks == 1) {
                const float by = l == 0.0f ? 0.0f : 1.0f / l;  // no key seen: zeros
                const uint32_t whole_row = row0 + row;
                uint16_t* to = a.out + (uint64_t)(n.first + whole_row / group) * a.out_stride +
                               (uint64_t)(kv * group + whole_row % group) * D + d0;
#pragma unroll
                for (int x = 0; x < D / 16; ++x) to[x] = __builtin_bit_cast(uint16_t, (__bf16)(o[x] * by));
            } else {
                float* to = part + row * D + d0;
#pragma unroll
                for (int x = 0; x < D / 16; ++x) to[x] = o[x];
                if (tid % 16 == 0) {
                    part[slot_rows * D + 2 * row] = fmaxf(fmaxf(tops[0][row], tops[1][row]), fmaxf(tops[2][row], tops[3][row]));
                    part[slot_rows * D + 2 * row + 1] = l;
                }
            }
        }
    }
}

// A wave a (token, q head): the chunks' partial rows against their largest maximum,
// in the order of the chunks.
template <int D>
__global__ __launch_bounds__(256) void join_kernel(AttentionArgs a, Split split, uint32_t slot_rows) {
    constexpr int E = D / 64;
    const uint32_t lane = threadIdx.x & 63, t = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (h >= a.q_heads) return;
    const uint32_t s = sequence_of(a.step.start, a.step.seqs, t);
    if (s >= a.step.seqs) return;
    const uint32_t group = a.q_heads / a.cache.kv_heads, kv = h / group, room = table_room(a.step, a.cache.page_shift);
    Chunk c;
    if (!find_chunk(a.step, room, group, split, s, true, c) || c.chunks == 1) return;
    const Lengths n = lengths_of(a.step, s, room);
    if (t - n.first >= n.fresh) return;
    const uint32_t r = (t - n.first) * group + h % group, row = r % split.rows;
    const uint64_t stride = (uint64_t)a.cache.kv_heads * slot_rows * (D + 2);
    const float* part = a.part + ((uint64_t)(c.slot + (c.blocks - 1 - r / split.rows) * c.chunks) * a.cache.kv_heads + kv) * slot_rows * (D + 2);
    const float* stats = part + slot_rows * D + 2 * row;
    float top = kNoMax;
    for (uint32_t i = lane; i < c.chunks; i += 64) top = fmaxf(top, stats[i * stride]);
#pragma unroll
    for (int off = 1; off < 64; off *= 2) top = fmaxf(top, __shfl_xor(top, off));
    float o[E] = {}, l = 0.0f;
    for (uint32_t i = 0; i < c.chunks; ++i) {
        const float w = __builtin_amdgcn_exp2f(stats[i * stride] - top);
        l = __builtin_fmaf(w, stats[i * stride + 1], l);
#pragma unroll
        for (int x = 0; x < E; ++x) o[x] = __builtin_fmaf(w, part[i * stride + row * D + lane * E + x], o[x]);
    }
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* to = a.out + t * a.out_stride + (uint64_t)h * D + lane * E;
#pragma unroll
    for (int x = 0; x < E; ++x) to[x] = __builtin_bit_cast(uint16_t, (__bf16)(o[x] * by));
}

template <int D, int NT>
hipError_t launch_rows(const AttentionArgs& a, uint32_t upto, int cus) {
    const uint32_t group = a.q_heads / a.cache.kv_heads, kv = a.cache.kv_heads;
    const uint32_t rows = a.step.max_tokens * group < upto ? a.step.max_tokens * group : upto;
    const uint32_t blocks = (rows + 16 * NT - 1) / (16 * NT), slot_rows = rows < 16 * NT ? rows : 16 * NT;
    // a cut row block has at least two chunks, so at most twice `target` chunks of a head need a slot
    const uint64_t slots = a.part_bytes / ((uint64_t)slot_rows * (D + 2) * 4);
    uint64_t target = 4ull * cus / kv;
    if (target > slots / 2 / kv) target = slots / 2 / kv;
    if (target < 1) target = 1;
    const Split split{(uint32_t)target, 16 * NT, 0, upto};
    const dim3 grid((uint32_t)target + a.step.seqs * blocks, kv);
    attention_rows_kernel<D, NT><<<grid, dim3(256), 0, a.stream>>>(a, split, slot_rows);
    return launch_join(a, split, slot_rows);
}

}  // namespace

hipError_t launch_join(const AttentionArgs& a, const Split& split, uint32_t slot_rows) {
    // (a table of one unit's pages holds no sequence that could be cut)
    if ((uint64_t)a.step.table_stride << a.cache.page_shift > kUnit && split.target > 1) {
        const dim3 grid(a.step.tokens, (a.q_heads + 3) / 4);
        if (a.cache.head_dim == 64) join_kernel<64><<<grid, dim3(256), 0, a.stream>>>(a, split, slot_rows);
        if (a.cache.head_dim == 128) join_kernel<128><<<grid, dim3(256), 0, a.stream>>>(a, split, slot_rows);
        if (a.cache.head_dim == 256) join_kernel<256><<<grid, dim3(256), 0, a.stream>>>(a, split, slot_rows);
    }
    return hipGetLastError();
}

// Sequences of up to 128 rows a kv head are bound by reading their keys, longer ones
// by the products.
constexpr uint32_t kFewRows = 128;

hipError_t launch_attention(const AttentionArgs& a, int cus) {
    const uint64_t rows = (uint64_t)a.step.max_tokens * (a.q_heads / a.cache.kv_heads);
    const bool many = rows > kFewRows;
    // (a step whose sequences all have max_tokens has none of the short kind)
    if (!many || (uint64_t)a.step.seqs * a.step.max_tokens != a.step.tokens) {
        const uint32_t most = many ? kFewRows : (uint32_t)rows;
        hipError_t e = hipSuccess;
#define MX4_ROWS(D)                                                        \
    if (a.cache.head_dim == D) {                                           \
        if (most <= 16) e = launch_rows<D, 1>(a, most, cus);               \
        else if (most <= 32 || D == 256) e = launch_rows<D, 2>(a, most, cus); \
        else e = launch_rows<D, D == 256 ? 2 : 4>(a, most, cus);           \
    }
        MX4_ROWS(64)
        MX4_ROWS(128)
        MX4_ROWS(256)
#undef MX4_ROWS
        if (e != hipSuccess || !many) return e;
    }
    return launch_attention_tiles(a, kFewRows, cus);
}

}  // namespace mx4
