// attention_tiles.hip -- attention of prompts: sequences with many query rows a kv
// head, where the products bound the time. (The mathematics: attention.hip.)
#include <hip/hip_runtime.h>

#include "attention_device.h"

namespace mx4 {

namespace {

constexpr uint32_t kTile = 64;  // keys in LDS at a time
constexpr uint32_t kNoRow = 0xffffffffu;

// K tile: row of D values a key, its 16-byte pieces xored by the key, so that the
// 16 keys that one read phase takes at one piece lie in 16 different places.
template <int D>
__device__ __forceinline__ uint32_t k_at(uint32_t key, uint32_t piece) {
    return key * D + ((piece ^ (D == 64 ? (key >> 1) & 7 : key & 15)) * 8);
}
// V^T tile: row of 64 keys a channel. The 16 keys of a product stand in the order in
// which its other operand, the weights, leaves the first product: lane half h, then
// key / 8, then key % 4. Pieces xored, and rows swapped in pairs, by the channel, for
// the reads (16 neighbouring channels, one piece) and the writes (every 8th channel).
__device__ __forceinline__ uint32_t v_at(uint32_t d, uint32_t piece) {
    return (d ^ ((d >> 3) & 1)) * kTile + ((piece ^ ((d >> 1) & 7) ^ ((d >> 4) & 7)) * 8);
}

// The rows go to the output, or, cut, to their slot; then what was left out (found).
template <int D, int RT>
__device__ __forceinline__ void finish(const AttentionArgs& a, const Chunk& c, const Lengths& n, const f32x16 (&acc)[RT][D / 32],
                                       const float (&top)[RT], const float (&l)[RT], const uint32_t (&token)[RT], bool found,
                                       uint32_t* bad, uint32_t key0, uint32_t key_end, uint32_t row0, uint32_t wave, uint32_t kv,
                                       uint32_t slot_rows) {
    constexpr int MT = D / 32;
    const uint32_t lane = threadIdx.x & 63, n32 = lane & 31, h = lane >> 5;
    const uint32_t kvs = a.cache.kv_heads, group = a.q_heads / kvs;
    float* part = a.part + ((uint64_t)(c.slot + c.chunk) * kvs + kv) * slot_rows * (D + 2);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const float sum = l[t] + __shfl_xor(l[t], 32);
        const uint32_t row = (wave * RT + t) * 32 + n32, r = row0 + row;
        if (token[t] == kNoRow) continue;
        if (c.chunks == 1) {
            const float by = sum == 0.0f ? 0.0f : 1.0f / sum;  // no key seen: zeros
            uint16_t* to = a.out + (uint64_t)(n.first + r / group) * a.out_stride + (uint64_t)(kv * group + r % group) * D + h * 4;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    __bf16 o[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = (__bf16)(acc[t][m][x * 4 + i] * by);
                    *reinterpret_cast<uint2*>(to + m * 32 + x * 8) = __builtin_bit_cast(uint2, o);
                }
        } else {
            float* to = part + row * D + h * 4;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    *reinterpret_cast<float2*>(to + m * 32 + x * 8) = {acc[t][m][x * 4], acc[t][m][x * 4 + 1]};
                    *reinterpret_cast<float2*>(to + m * 32 + x * 8 + 2) = {acc[t][m][x * 4 + 2], acc[t][m][x * 4 + 3]};
                }
            if (h == 0) {
                part[slot_rows * D + 2 * row] = top[t];
                part[slot_rows * D + 2 * row + 1] = sum;
            }
        }
    }
    if (found) *bad = 1;
    __syncthreads();
    if (!*bad) return;
    for (uint32_t key = max(key0, n.before); key < key_end; ++key)
#pragma unroll 1
        for (int t = 0; t < RT; ++t) {
            const uint32_t row = (wave * RT + t) * 32 + n32, r = row0 + row;
            if (r < n.fresh * group)
#pragma unroll 1
                for (uint32_t e = 0; e < D / 2; ++e) add_to_stored(a, c, n, key, kv, r, row, e / 4 * 8 + h * 4 + e % 4, part);
        }
}

// A workgroup's way from the paged cache to the tiles: 64 keys' pieces in registers,
// then in LDS. Keys: 16-byte piece tid % PIECES of key tid / PIECES + i 256 / PIECES.
// Values: 4 keys of a wave's 16 by 8 channels, turned round by v_perm.
template <int D>
struct Stage {
    static constexpr int PIECES = D / 8, KLOADS = kTile * PIECES / 256, VROUNDS = PIECES > 16 ? PIECES / 16 : 1;
    const uint16_t *k, *v;
    const uint32_t* table;
    uint32_t table_last, page_last, kvs, kv, shift, wave, tid;
    uint32_t pages, pages_next, pages_at;  // lane i: page of 16-key group 4 pages_at + i, and of the 64 groups after
    u32x4 kr[KLOADS], vr[VROUNDS][4];

    __device__ __forceinline__ uint32_t look_up(uint32_t tile) const {
        return min(table[min((tile * 4 + (tid & 63)) << 4 >> shift, table_last)], page_last);
    }
    __device__ __forceinline__ void begin(uint32_t tile) {
        pages_at = tile;
        pages = look_up(tile);
        pages_next = look_up(tile + 16);
    }
    __device__ __forceinline__ uint64_t group_at(uint32_t tile, uint32_t group) const {  // elements
        const uint32_t page = __builtin_amdgcn_readlane(pages, (tile - pages_at) * 4 + group);
        return ((((uint64_t)page * kvs + kv) << shift) + ((tile * kTile + group * 16) & ((1u << shift) - 1))) * D;
    }
    __device__ __forceinline__ void load(uint32_t tile) {
        if (tile - pages_at == 16) {
            pages_at = tile;
            pages = pages_next;
            pages_next = look_up(tile + 16);
        }
#pragma unroll
        for (int i = 0; i < KLOADS; ++i) {
            const uint32_t key = (i * 256 + wave * 64) / PIECES;  // the wave's first: all its keys are in one group
            const uint16_t* from = k + group_at(tile, key / 16);
            kr[i] = *reinterpret_cast<const u32x4*>(from + ((key & 15) + (tid & 63) / PIECES) * D + (tid & 63) % PIECES * 8);
        }
        const uint16_t* from = v + group_at(tile, wave);
        const uint32_t lane = tid & 63, vc = PIECES >= 16 ? lane & 15 : lane & 7, va = PIECES >= 16 ? lane >> 4 : (lane >> 3) & 3;
#pragma unroll
        for (int e = 0; e < VROUNDS; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) vr[e][i] = *reinterpret_cast<const u32x4*>(from + (va * 4 + i) * D + (e * 16 + vc) * 8);
    }
    // edge: the tile may hold new tokens or keys that are not there. Those count as zeros; values
    // of new tokens that are not finite do so too here (found: there are some), the rows that
    // see them get them at the end.
    __device__ __forceinline__ void store(uint32_t tile, uint16_t* kbuf, uint16_t* vbuf, uint32_t before, uint32_t keys, bool& found) {
#pragma unroll
        for (int i = 0; i < KLOADS; ++i) {
            const uint32_t p = i * 256 + tid;
            *reinterpret_cast<u32x4*>(&kbuf[k_at<D>(p / PIECES, p % PIECES)]) = kr[i];
        }
        const uint32_t lane = tid & 63, vc = PIECES >= 16 ? lane & 15 : lane & 7, va = PIECES >= 16 ? lane >> 4 : (lane >> 3) & 3;
        if (tile * kTile + kTile > before) {
            const uint32_t key = tile * kTile + wave * 16 + va * 4;
#pragma unroll
            for (int e = 0; e < VROUNDS; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        uint32_t w = key + i < keys ? vr[e][i][x] : 0u;
                        found |= not_finite(w);
                        vr[e][i][x] = finite_only(w);
                    }
        }
        if (PIECES >= 16 || lane < 32) {
            const uint32_t piece = wave * 2 + (va & 1), part = (va >> 1) * 4;
#pragma unroll
            for (int e = 0; e < VROUNDS; ++e)
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const uint32_t sel = x % 2 ? 0x07060302u : 0x05040100u;
                    const uint2 w = {__builtin_amdgcn_perm(vr[e][1][x / 2], vr[e][0][x / 2], sel),
                                     __builtin_amdgcn_perm(vr[e][3][x / 2], vr[e][2][x / 2], sel)};
                    *reinterpret_cast<uint2*>(&vbuf[v_at((e * 16 + vc) * 8 + x, piece) + part]) = w;
                }
        }
    }
};

// Four waves, each with RT tiles of 32 rows against the workgroup's keys, 64 at a
// time in LDS (the next 64 on their way in registers). S^T = K Q^T in 32 x 32 x 16
// products leaves lane (row n = lane % 32, half h) the scores of keys 8 b + 4 h + i;
// packed in that order they are the operand P^T of O^T = V^T P^T.
template <int D, int RT>
__global__ __launch_bounds__(256, RT == 1 && D <= 128 ? 2 : 1) void attention_tiles_kernel(AttentionArgs a, Split split,
                                                                                           uint32_t slot_rows) {
    constexpr int KK = D / 16, MT = D / 32;
    __shared__ __align__(16) uint16_t kbuf[2][kTile * D];
    __shared__ __align__(16) uint16_t vbuf[2][kTile * D];
    __shared__ uint32_t bad;
    const uint32_t tid = threadIdx.x, lane = tid & 63, n32 = lane & 31, h = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t kvs = a.cache.kv_heads, kv = blockIdx.x % kvs, group = a.q_heads / kvs, shift = a.cache.page_shift;
    const uint32_t room = table_room(a.step, shift);
    Chunk c;
    if (!find_chunk(a.step, room, group, split, blockIdx.x / kvs, false, c)) return;
    const uint32_t seq = __builtin_amdgcn_readfirstlane(c.s);
    const Lengths n = lengths_of(a.step, seq, room);
    const uint32_t row0 = c.block * (128 * RT), all_rows = n.fresh * group;
    // chains: the keys that the block's last row sees; and how far all rows of the block see
    const uint32_t last_row = min(row0 + 128 * RT, all_rows) - 1;
    const uint32_t end_key = a.tree ? n.keys : min(n.keys, n.before + last_row / group + 1);
    const uint32_t clear = a.tree ? n.before : min(n.keys, n.before + row0 / group + 1);
    const uint32_t tile0 = __builtin_amdgcn_readfirstlane(c.chunk * c.cu * (kUnit / kTile));
    const uint32_t tile_end =
        __builtin_amdgcn_readfirstlane(min(tile0 + c.cu * (kUnit / kTile), (end_key + kTile - 1) / kTile));
    Stage<D> st;
    st.k = a.cache.k;
    st.v = a.cache.v;
    st.table = a.step.table + (uint64_t)seq * a.step.table_stride;
    st.table_last = a.step.table_stride - 1;
    st.page_last = a.cache.pages - 1;
    st.kvs = kvs;
    st.kv = kv;
    st.shift = shift;
    st.wave = wave;
    st.tid = tid;
    if (tile0 < tile_end) {
        st.begin(tile0);
        st.load(tile0);
    }

    bf16x8 q[RT][KK];
    uint32_t token[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const uint32_t r = row0 + (wave * RT + t) * 32 + n32;
        token[t] = r < all_rows ? r / group : kNoRow;
        const uint16_t* from = a.q + (uint64_t)(n.first + r / group) * a.q_stride + (uint64_t)(kv * group + r % group) * D + h * 8;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            u32x4 w = {0, 0, 0, 0};
            if (token[t] != kNoRow) w = *reinterpret_cast<const u32x4*>(from + kk * 16);
            q[t][kk] = __builtin_bit_cast(bf16x8, w);
        }
    }
    const float cs = a.scale * 1.44269504088896340736f;

    f32x16 acc[RT][MT];
    float top[RT], l[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        top[t] = kNoMax;
        l[t] = 0.0f;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int x = 0; x < 16; ++x) acc[t][m][x] = 0.0f;
    }
    bool found = false;
    if (tid == 0) bad = 0;
    if (tile0 < tile_end) st.store(tile0, kbuf[0], vbuf[0], n.before, n.keys, found);
    for (uint32_t tile = tile0; tile < tile_end; ++tile) {
        const uint32_t b = (tile - tile0) & 1;
        __syncthreads();
        if (tile + 1 < tile_end) st.load(tile + 1);
        const bool whole = tile * kTile + kTile <= clear;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            f32x16 s[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int x = 0; x < 16; ++x) s[t][x] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                const bf16x8 kf = *reinterpret_cast<const bf16x8*>(&kbuf[b][k_at<D>(sub * 32 + n32, kk * 2 + h)]);
#pragma unroll
                for (int t = 0; t < RT; ++t) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, q[t][kk], s[t], 0, 0, 0);
            }
            bf16x8 p[RT][2];
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                if (!whole) {
                    const uint32_t seen = token[t] != kNoRow ? seen_window(a, n, token[t], tile * kTile + sub * 32) : 0u;
#pragma unroll
                    for (int x = 0; x < 16; ++x)
                        if (!(seen >> (x / 4 * 8 + h * 4 + x % 4) & 1)) s[t][x] = -INFINITY;
                }
                float most = s[t][0];
#pragma unroll
                for (int x = 1; x < 16; ++x) most = fmaxf(most, s[t][x]);
                most *= cs;
                if (__any(most > top[t] + kSlack)) {
                    most = fmaxf(most, __shfl_xor(most, 32));
                    const float now = fmaxf(top[t], most), keep = __builtin_amdgcn_exp2f(top[t] - now);
                    top[t] = now;
                    l[t] *= keep;
#pragma unroll
                    for (int m = 0; m < MT; ++m) acc[t][m] *= keep;
                }
#pragma unroll
                for (int x = 0; x < 16; ++x)
                    p[t][x / 8][x % 8] = (__bf16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[t][x], cs, -top[t]));
                const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
                for (int x = 0; x < 8; ++x)  // of the rounded weights
                    l[t] = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{p[t][x / 4][x % 4 * 2], p[t][x / 4][x % 4 * 2 + 1]}, one, l[t], false);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const bf16x8 vt = *reinterpret_cast<const bf16x8*>(&vbuf[b][v_at(m * 32 + n32, sub * 4 + u * 2 + h)]);
#pragma unroll
                    for (int t = 0; t < RT; ++t) acc[t][m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vt, p[t][u], acc[t][m], 0, 0, 0);
                }
        }
        if (tile + 1 < tile_end) st.store(tile + 1, kbuf[b ^ 1], vbuf[b ^ 1], n.before, n.keys, found);
    }
    finish<D, RT>(a, c, n, acc, top, l, token, found, &bad, tile0 * kTile, min(tile_end * kTile, n.keys), row0, wave, kv,
                  slot_rows);
}

template <int D, int RT>
hipError_t launch_tiles(const AttentionArgs& a, uint32_t over, int cus) {
    constexpr uint32_t ROWS = 128 * RT;
    const uint32_t group = a.q_heads / a.cache.kv_heads, kv = a.cache.kv_heads;
    const uint64_t rows = (uint64_t)a.step.max_tokens * group;
    // row blocks of a kv head: the tokens' whole ones, and a partial one a sequence
    const uint64_t whole = (uint64_t)a.step.tokens * group / ROWS, blocks = whole + a.step.seqs;
    const uint32_t slot_rows = rows < ROWS ? (uint32_t)rows : ROWS;
    // enough row blocks to fill the CUs several times over need no cutting
    const uint64_t wanted = whole * kv >= 4ull * cus ? 1 : 2ull * cus / kv;
    const Split split{split_target(a, wanted, blocks, slot_rows), ROWS, over, 0xffffffffu};
    attention_tiles_kernel<D, RT><<<dim3((uint32_t)((split.target + blocks) * kv)), dim3(256), 0, a.stream>>>(a, split, slot_rows);
    return launch_join(a, split, blocks, slot_rows);
}

}  // namespace

hipError_t launch_attention_tiles(const AttentionArgs& a, uint32_t over, int cus) {
    if (a.cache.head_dim == 64) return launch_tiles<64, 1>(a, over, cus);
    if (a.cache.head_dim == 128) return launch_tiles<128, 1>(a, over, cus);
    return launch_tiles<256, 1>(a, over, cus);
}

}  // namespace mx4
