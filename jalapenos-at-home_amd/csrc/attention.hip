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

#include "cache_device.h"

namespace mx4 {

namespace {

constexpr float kNoMax = -3.4028234664e38f;  // below every score: 2^(s - kNoMax) is never taken, -inf - kNoMax = -inf
// A row's maximum is raised only when a score passes it by this much: weights stay
// below 2^8, their sums far inside f32, and most steps leave the accumulators alone.
constexpr float kSlack = 8.0f;
constexpr uint32_t kUnit = 128;  // keys: the grain in which a sequence is cut among workgroups

// ------------------------------------------------------------- the split along the keys

// How the step's work is cut. Every (row block, kv head) of a sequence has
// ceil(units / cu) chunks of cu units; cu makes about `target` chunks a kv head of
// the whole step, from the lengths in device memory. Chunks of cut rows leave
// partial results in slots, joined by join_kernel.
struct Chunk {
    uint32_t s, block, chunk, chunks, slot, cu;  // slot: of the row block's first chunk, a kv head's numbering
};

struct Lengths {
    uint32_t first, fresh, before, keys;
};

__device__ __forceinline__ Lengths lengths_of(const StepView& st, uint32_t s, uint32_t room) {
    Lengths n;
    tokens_of(st, s, n.first, n.fresh);
    n.before = min(st.cached[s], room);
    n.keys = min(n.before + n.fresh, room);
    return n;
}

__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
#pragma unroll
    for (int off = 1; off < 64; off *= 2) v += __shfl_xor(v, off);
    return v;
}

__device__ __forceinline__ uint32_t wave_prefix(uint32_t v) {  // inclusive
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
        const uint32_t o = __shfl_up(v, off);
        v += lane >= (uint32_t)off ? o : 0;
    }
    return v;
}

// The chunk that is number `item` of its kv head, or (by_sequence) the first one of
// sequence `item`'s row block 0. False: there is none. Called by whole waves.
__device__ __forceinline__ bool find_chunk(const StepView& st, uint32_t room, uint32_t group, uint32_t rows, uint32_t target,
                                           uint32_t item, bool by_sequence, Chunk& c) {
    const uint32_t lane = threadIdx.x & 63;
    auto shape = [&](uint32_t s, uint32_t& units, uint32_t& blocks) {
        units = blocks = 0;
        if (s >= st.seqs) return;
        const Lengths n = lengths_of(st, s, room);
        if (n.fresh == 0) return;
        units = max((n.keys + kUnit - 1) / kUnit, 1u);
        blocks = (n.fresh * group + rows - 1) / rows;
    };
    uint32_t total = 0;
    for (uint32_t s0 = 0; s0 < st.seqs; s0 += 64) {
        uint32_t units, blocks;
        shape(s0 + lane, units, blocks);
        total += wave_sum(units * blocks);
    }
    c.cu = max((total + target - 1) / target, 1u);
    uint32_t items = 0, slots = 0;
    for (uint32_t s0 = 0; s0 < st.seqs; s0 += 64) {
        uint32_t units, blocks;
        shape(s0 + lane, units, blocks);
        const uint32_t chunks = (units + c.cu - 1) / c.cu, mine = chunks * blocks, cut = chunks > 1 ? mine : 0;
        const uint32_t upto = items + wave_prefix(mine), slots_upto = slots + wave_prefix(cut);
        const uint64_t hit = by_sequence ? (item - s0 < 64 ? 1ull << (item - s0) : 0ull) : __ballot(item < upto);
        if (hit) {
            const int at = __ffsll((unsigned long long)hit) - 1;
            c.s = s0 + at;
            c.chunks = __shfl(chunks, at);
            const uint32_t in = by_sequence ? 0 : item - (__shfl(upto, at) - __shfl(mine, at));
            if (c.chunks == 0) return false;
            c.block = in / c.chunks;
            c.chunk = in % c.chunks;
            c.slot = __shfl(slots_upto, at) - __shfl(cut, at) + c.block * c.chunks;
            return true;
        }
        items = __shfl(upto, 63);
        slots = __shfl(slots_upto, 63);
    }
    return false;
}

// ------------------------------------------------------------- few rows a sequence

// The keys that row (first + i) sees of the 32 from k0 on, one bit each.
__device__ __forceinline__ uint32_t seen_window(const AttentionArgs& a, const Lengths& n, uint32_t i, uint32_t k0) {
    const int64_t j0 = (int64_t)k0 - n.before;  // place among the new tokens
    const int64_t most = (int64_t)n.keys - k0;  // keys that there are
    const uint32_t there = most >= 32 ? ~0u : most <= 0 ? 0u : (1u << most) - 1;
    if (!a.tree) {
        const int64_t sees = (int64_t)i + 1 - j0;
        return there & (sees >= 32 ? ~0u : sees <= 0 ? 0u : (1u << sees) - 1);
    }
    const uint64_t* row = a.tree + (uint64_t)(n.first + i) * a.tree_words;
    auto word = [&](int64_t w) { return w < 0 ? ~0ull : w < a.tree_words ? row[w] : 0ull; };
    const int64_t w = j0 >> 6;
    const uint32_t shift = (uint32_t)(j0 & 63);
    uint64_t bits = word(w) >> shift;
    if (shift > 32) bits |= word(w + 1) << (64 - shift);
    return there & (uint32_t)bits;
}

__device__ __forceinline__ bool not_finite(uint32_t pair) {  // either bf16 of a word
    return (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u;
}

// A workgroup's four waves take the chunk's steps of 32 keys in turn, each with all
// 16 NT rows, keys and values straight from memory to registers. S^T = K Q^T
// leaves lane (row n = lane % 16, group g = lane / 16) the scores of keys 4 g .. 4 g + 3
// of each half step, which is what the next product's operand P^T wants from it if the
// values come in the same order -- so weights never cross lanes. A lane loads the 8 keys
// of its group at 8 neighbouring channels, and the 8 x 8 block turned round in
// registers (one v_perm a word) serves as the operand V^T of 8 products, channel
// 8 (lane % 16) + m in the m-th.
template <int D, int NT>
__global__ __launch_bounds__(256, NT <= 2 && D <= 128 ? 2 : 1) void attention_rows_kernel(AttentionArgs a, uint32_t target,
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
    if (!find_chunk(a.step, room, group, ROWS, target, blockIdx.x, false, c)) return;
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
                        if ((vf[j][x] & 0x7f80u) == 0x7f80u) vf[j][x] &= 0xffff0000u;
                        if ((vf[j][x] & 0x7f800000u) == 0x7f800000u) vf[j][x] &= 0xffffu;
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
__global__ __launch_bounds__(256) void join_kernel(AttentionArgs a, uint32_t target, uint32_t slot_rows, uint32_t block_rows) {
    constexpr int E = D / 64;
    const uint32_t lane = threadIdx.x & 63, t = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (h >= a.q_heads) return;
    const uint32_t s = sequence_of(a.step.start, a.step.seqs, t);
    if (s >= a.step.seqs) return;
    const uint32_t group = a.q_heads / a.cache.kv_heads, kv = h / group, room = table_room(a.step, a.cache.page_shift);
    Chunk c;
    if (!find_chunk(a.step, room, group, block_rows, target, s, true, c) || c.chunks == 1) return;
    const Lengths n = lengths_of(a.step, s, room);
    if (t - n.first >= n.fresh) return;
    const uint32_t r = (t - n.first) * group + h % group, row = r % block_rows;
    const uint64_t stride = (uint64_t)a.cache.kv_heads * slot_rows * (D + 2);
    const float* part = a.part + ((uint64_t)(c.slot + r / block_rows * c.chunks) * a.cache.kv_heads + kv) * slot_rows * (D + 2);
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
hipError_t launch_rows(const AttentionArgs& a, int cus) {
    const uint32_t group = a.q_heads / a.cache.kv_heads, rows = a.step.max_tokens * group, kv = a.cache.kv_heads;
    const uint32_t blocks = (rows + 16 * NT - 1) / (16 * NT), slot_rows = rows < 16 * NT ? rows : 16 * NT;
    // a cut row block has at least two chunks, so at most twice `target` chunks of a head need a slot
    const uint64_t slots = a.part_bytes / ((uint64_t)slot_rows * (D + 2) * 4);
    uint64_t target = 4ull * cus / kv;
    if (target > slots / 2 / kv) target = slots / 2 / kv;
    if (target < 1) target = 1;
    const dim3 grid((uint32_t)target + a.step.seqs * blocks, kv);
    attention_rows_kernel<D, NT><<<grid, dim3(256), 0, a.stream>>>(a, (uint32_t)target, slot_rows);
    // (a table of one unit's pages holds no sequence that could be cut)
    if ((uint64_t)a.step.table_stride << a.cache.page_shift > kUnit)
        join_kernel<D><<<dim3(a.step.tokens, (a.q_heads + 3) / 4), dim3(256), 0, a.stream>>>(a, (uint32_t)target, slot_rows, 16 * NT);
    return hipGetLastError();
}

}  // namespace

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
    const uint64_t rows = (uint64_t)a.step.max_tokens * (a.q_heads / a.cache.kv_heads);
    if (rows <= 128) {
#define MX4_ROWS(D)                                                       \
    if (a.cache.head_dim == D) {                                          \
        if (rows <= 16) return launch_rows<D, 1>(a, cus);                 \
        if (rows <= 32 || D == 256) return launch_rows<D, 2>(a, cus);     \
        return launch_rows<D, D == 256 ? 2 : 4>(a, cus);                  \
    }
        MX4_ROWS(64)
        MX4_ROWS(128)
        MX4_ROWS(256)
#undef MX4_ROWS
    }
    const dim3 grid(a.step.tokens, a.q_heads);
    if (a.cache.head_dim == 64) attention_kernel<64><<<grid, dim3(256), 0, a.stream>>>(a);
    if (a.cache.head_dim == 128) attention_kernel<128><<<grid, dim3(256), 0, a.stream>>>(a);
    if (a.cache.head_dim == 256) attention_kernel<256><<<grid, dim3(256), 0, a.stream>>>(a);
    return hipGetLastError();
}

}  // namespace mx4
