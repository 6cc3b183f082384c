// Cache attention in 16 bits, heads of up to 256, few rows (attend_item): single
// tokens above all.
//
// Scores are S^T = K Q^T on 16x16x32 MFMAs (keys on the M axis): lane (j = lane %
// 16, g = lane / 16) ends with S[row j][key 4 g + i], i < 4, of each half of a
// 32-key tile, which is the operand layout that the product O^T += V^T P^T takes its
// weights in (its key order then is 4 g .. 4 g + 3 of one half and of the other),
// so they never change lanes.  The four wavefronts stream tiles of their own: K from
// memory straight into the MFMA operand, a lane 16 bytes of its key's row; V in
// whole rows into registers and through a tile of LDS of the wavefront's own, to be
// read transposed (ds_read_b64_tr_b16: in a 16-lane group, lane i receives element
// i % 4 of the 8-byte pieces that lanes 4 e + i / 4 read).  Registers are refilled
// as soon as their tile is used, so that 16 KiB of a wavefront (dim 128) are always
// under way, without a barrier.
//
// Bound by memory: a batch of 64 sequences of up to 8,192 keys, 8 kv heads of
// 128, is read at 5.2 TB/s in 214 us (a copy of 2 GB runs at 4.8).
#pragma once

#include "xattn_cache_item.h"

namespace xattn {
namespace cache {

template <typename T, int D>
struct FewShape {
    static constexpr int kKeys = 32;              // keys of a tile
    static constexpr int kRegs = D / 16;          // 16-byte registers of a lane for K, for V
    static constexpr int kBlocks = D / 16;        // 16-column blocks of the output
    static constexpr int kPieces = D / 8;         // 16-byte pieces of a row
    static constexpr int kVRow = D * 2 + 32;      // bytes of a V row in LDS: 32 of padding deal
                                                  // four rows to distinct banks
    static constexpr int kVTile = kKeys * kVRow;
    static constexpr int kORow = D + 4;           // floats of an output row in LDS
    static constexpr int kWaveLds =
        kVTile > kRows * kORow * 4 ? kVTile : kRows * kORow * 4;
    static constexpr int kStats = kWaves * kRows * 8;  // maxima and sums
    static constexpr int kLds = kWaves * kWaveLds + kStats;
};

template <typename T, int D, bool PREFIX>
__device__ __forceinline__ void attend_item(const AttendParams& p, unsigned block, char* lds) {
    typedef FewShape<T, D> S;
    constexpr int KT = S::kKeys, NR = S::kRegs, NB = S::kBlocks;
    float2(*const stats)[kRows] = (float2(*)[kRows])(lds + kWaves * S::kWaveLds);
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int j = lane % 16, g = lane / 16;

    Item it;
    if (!find_item<kRows, PREFIX>(p, block, &it)) return;
    const Sequence& s = it.s;
    const int least = it.least, k0 = it.k0, k1 = it.k1;

    // Lane j's row.  Rows behind the last repeat it and are not stored.
    const Row mine = it.row(p, min(j, it.rows - 1));
    const int seen[1] = {min(s.seen(mine.token, it.causal), k1)};
    u4 qr[NR / 2];
    {
        const T* q = (const T*)p.q + mine.token * p.qs + (long long)mine.head * D + 8 * g;
#pragma unroll
        for (int r = 0; r < NR / 2; ++r) qr[r] = *(const u4*)(q + 32 * r) ^ p.sign;
    }

    f4 o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = f4{0, 0, 0, 0};
    float m[1] = {-INFINITY}, l[1] = {0.0f}, keep[1];
    bool bad = false, odd = false;

    // Rows of the cache that a tile's keys lie on: lane's key is k + lane % KT.
    struct Where {
        int id;
        unsigned slot;
    };
    const auto find = [&](int k) {
        const unsigned key = (unsigned)min(k + lane % KT, k1 - 1);
        const unsigned page = p.pages.page_size.div(key);
        return Where{it.table[page], key - page * p.pages.page_size.d};
    };
    const auto row_of = [&](const Where& w) {
        const bool ok = w.id >= 0 && (unsigned)w.id < p.pages.num_pages;
        bad |= !ok;
        return ((ok ? (unsigned)w.id : 0u) * p.pages.kv_heads + it.kv_head) *
                   p.pages.page_size.d + w.slot;
    };
    u4 kr[NR], vr[NR];
    const auto load_k = [&](unsigned row) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const char* a = p.pages.k + (size_t)__shfl(row, 16 * h + j) * (D * 2) + 16 * g;
#pragma unroll
            for (int r = 0; r < NR / 2; ++r) kr[h * NR / 2 + r] = *(const u4*)(a + 64 * r);
        }
    };
    // V register r of a lane is piece 64 r + lane of the tile in row order.
    const auto v_row = [&](int r) { return 64 / S::kPieces * r + lane / S::kPieces; };
    const int v_piece = lane % S::kPieces;
    const auto load_v = [&](unsigned row) {
#pragma unroll
        for (int r = 0; r < NR; ++r)
            vr[r] = *(const u4*)(p.pages.v + (size_t)__shfl(row, v_row(r)) * (D * 2) +
                                 16 * v_piece);
    };

    char* const vt = lds + wave * S::kWaveLds;
    const int step = kWaves * KT;
    int k = k0 + wave * KT;
    if (k < k1) {
        Where next = find(k);
        const unsigned row = row_of(next);
        next = find(k + step);
        load_k(row);
        load_v(row);
        for (; k < k1; k += step) {
            const bool more = k + step < k1;
            const Where after = find(k + 2 * step);
            f4 sc[1][2];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const int h = r % 2, i = r / 2;
                sc[0][h] = mfma32<T>(kr[h * NR / 2 + i], qr[i], i ? sc[0][h] : f4{0, 0, 0, 0});
            }
            unsigned next_row = 0;
            if (more) {
                next_row = row_of(next);
                load_k(next_row);
            }
            next = after;
            const bool partial = k + KT > least;  // some row does not see all of the tile
            if (weights(p, sc, partial, k + 4 * g, seen, m, l, keep))
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] *= keep[0];
            if (partial)
#pragma unroll
                for (int r = 0; r < NR; ++r) odd |= clear_not_finite<T>(vr[r]);
#pragma unroll
            for (int r = 0; r < NR; ++r) *(u4*)(vt + v_row(r) * S::kVRow + 16 * v_piece) = vr[r];
            if (more) load_v(next_row);
            const u4 w = pack8<T>(sc[0][0], sc[0][1]);
            const char* from = vt + (4 * g + j / 4) * S::kVRow + j % 4 * 8;
#pragma unroll
            for (int b = 0; b < NB; ++b)
                o[b] = mfma32<T>(transposed(from + 32 * b, from + 32 * b + 16 * S::kVRow), w, o[b]);
        }
    }
    if (__ballot(odd))
        for (int t = k0 + wave * KT; t < k1; t += step)
            for (int c = t; t + KT > least && c < min(t + KT, k1); ++c)
                if (const char* v = it.row_of_v(p, c, D * 2))
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const f4 x = odd_values<T>(v + (16 * b + 4 * g) * 2);
                        if (c < seen[0]) o[b] += x;
                    }
    float sum = wave_sum16_groups(l[0]);
    if (__ballot(bad)) sum = NAN;
    if (lane < kRows) stats[wave][lane] = {m[0] * p.c2, sum};
    float* part = (float*)vt + j * S::kORow;
#pragma unroll
    for (int b = 0; b < NB; ++b) *(f4*)(part + 16 * b + 4 * g) = o[b];
    __syncthreads();
    join_and_store<T, D, PREFIX, kRows>(p, it, stats, lds, S::kWaveLds, S::kORow);
}

}  // namespace cache
}  // namespace xattn
