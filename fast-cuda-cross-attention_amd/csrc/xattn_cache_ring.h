// Cache attention in 16 bits at dim 768 (ring_item): RB blocks of sixteen rows, one or
// two.
//
// Operands, scores and weights as in xattn_cache_few.h.  The four wavefronts share
// tiles of 32 keys and own 192 columns each, of Q, K, V and the output; their shares
// of the scores are summed through LDS, one barrier a tile.
//
// K arrives by DMA in a slice of LDS of the wavefront's own: straight into the
// operand's layout, whose neighbouring lanes are different rows, a KiB would hold
// the CU's path to memory for 64 cycles instead of 16.  Its pieces are swizzled so
// that neighbouring rows use distinct banks.  V comes in whole rows into registers
// and passes through LDS to be read transposed.
//
// A tile's scores come before the product of the tile before it with V, under which
// the next K is asked for, piece by piece, and the shares of the scores are
// exchanged; then V of this tile is asked for, and its softmax done.  So everything
// that arrives has a product's time or more to do so, and LDS need hold one K.
//
// Bound by that path: a tile of K and V is 96 KiB, 1,536 cycles, against 384 RB of
// matrix instructions.  32 sequences of 4,000 keys, one token each, are read at
// 4.9 TB/s; 64 rows over 50,176 keys take 69 us with two blocks and 79 with one.
#pragma once

#include "xattn_cache_item.h"

namespace xattn {
namespace cache {

template <int RB>
struct RingShape {
    static constexpr int kDW = kDim / kWaves;           // columns of a wavefront
    static constexpr int kKeys = 32;                    // keys of a tile
    static constexpr int kRegs = kDW / 16;              // KiB of a wavefront's K, or V, in a tile
    static constexpr int kBlocks = kDW / 16;            // 16-column blocks of the output
    static constexpr int kRow = kDW * 2;                // bytes of a row's columns
    static constexpr int kPieces = kRow / 16;
    // A KiB holds 64 pieces of consecutive rows; kPeriod KiB hold kStep whole rows.
    static constexpr int kPeriod = 3, kStep = 8;
    static_assert(kPeriod * 64 == kStep * kPieces, "whole rows");
    static constexpr int kKTile = kRegs * 1024;
    static constexpr int kVRow = kRow + 32;             // in LDS; 32 bytes of padding deal four
                                                        // rows to distinct banks
    static constexpr int kWaveLds = kKTile + kKeys * kVRow;
    static constexpr int kShare = RB * kKeys * kRows * 4;  // bytes of a wavefront's share of scores
    static constexpr int kLds = kWaves * kWaveLds + 2 * kWaves * kShare;
};

template <typename T, int RB, bool PREFIX>
__device__ __forceinline__ void ring_item(const AttendParams& p, unsigned block, char* lds) {
    typedef RingShape<RB> S;
    constexpr int KT = S::kKeys, KB = KT / 16, NR = S::kRegs, NB = S::kBlocks, NQ = NR / 2;
    constexpr int PERIOD = S::kPeriod, STEP = S::kStep, ROW = kDim * 2;
    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int j = lane % 16, g = lane / 16;

    Item it;
    if (!find_item<RB * kRows, PREFIX>(p, block, &it)) return;
    const Sequence& s = it.s;
    const int least = it.least, k0 = it.k0, k1 = it.k1;

    // Q: register r of lane (j, g) holds elements 32 r + 8 g .. + 7 of row j.
    const int col0 = wave * S::kDW;
    int seen[RB];
    u4 qr[RB][NQ];
    f4 o[RB][NB];
    float m[RB], l[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const Row mine = it.row(p, min(kRows * b + j, it.rows - 1));
        seen[b] = min(s.seen(mine.token, it.causal), k1);
        const T* q =
            (const T*)p.q + mine.token * p.qs + (long long)mine.head * kDim + col0 + 8 * g;
#pragma unroll
        for (int r = 0; r < NQ; ++r) qr[b][r] = *(const u4*)(q + 32 * r) ^ p.sign;
#pragma unroll
        for (int i = 0; i < NB; ++i) o[b][i] = f4{0, 0, 0, 0};
        m[b] = -INFINITY;
        l[b] = 0.0f;
    }
    bool bad = false, odd = false;

    // Where a tile's rows are.  Sixteen rows lie on one page where sixteen divides
    // the page size: their address is then one scalar plus a lane's constant offset; a
    // lane's own address otherwise, and where rows behind the last key repeat it.
    const unsigned size = p.pages.page_size.d;
    const bool runs = size % 16 == 0;
    const auto find = [&](int k) {  // lane's page: that of key k + lane % KT
        return it.table[p.pages.page_size.div((unsigned)min(k + lane % KT, k1 - 1))];
    };
    const auto row_at = [&](int page, unsigned key) {
        const bool ok = page >= 0 && (unsigned)page < p.pages.num_pages;
        bad |= !ok;
        return ((ok ? (unsigned)page : 0u) * p.pages.kv_heads + it.kv_head) * size +
               (key - p.pages.page_size.div(key) * size);
    };
    const auto halves = [&](int ids, int k, size_t (&from)[KB]) {  // byte offsets, scalars
#pragma unroll
        for (int h = 0; h < KB; ++h) {
            const unsigned row = row_at(__builtin_amdgcn_readlane(ids, 16 * h), k + 16 * h);
            from[h] = (size_t)row * ROW + col0 * 2;
        }
    };
    const auto one = [&](const char* pool, int ids, int k, int r) {  // row r
        const unsigned row = row_at(__shfl(ids, r), (unsigned)min(k + r, k1 - 1));
        return pool + (size_t)row * ROW + col0 * 2;
    };
    // (The lane read through an empty asm: what the rare paths derive from it is
    // otherwise kept in registers across the loop.)
    const auto hidden_lane = [&]() {
        int i = lane;
        asm volatile("" : "+v"(i));
        return i;
    };

    // K by DMA: KiB c of a tile.
    char* const kt = lds + wave * S::kWaveLds;
    const unsigned kt_at = __builtin_amdgcn_readfirstlane(lds_u32(kt));
    const auto swizzle = [](int row) { return row / 2 % 4 * 2; };
    int row_of[PERIOD], piece_of[PERIOD];
#pragma unroll
    for (int i = 0; i < PERIOD; ++i) {
        row_of[i] = (i * 64 + lane) / S::kPieces;
        piece_of[i] = (i * 64 + lane) % S::kPieces;
    }
    const DmaSrc pool = dma_base(p.pages.k);
    const auto k_whole = [&](const size_t (&from)[KB], int c) {
        const int row = STEP * (c / PERIOD), i = c % PERIOD;
        dma16_m0<0>(pool + (from[row / 16] + (size_t)(row % 16 * ROW)),
                    (unsigned)(row_of[i] * ROW + 16 * (piece_of[i] ^ swizzle(row + row_of[i]))),
                    kt_at + 1024 * c);
    };
    const auto k_any = [&](int ids, int k) {
        const int me = hidden_lane();
#pragma unroll
        for (int c = 0; c < NR; ++c) {
            const int i = c % PERIOD * 64 + me, row = STEP * (c / PERIOD) + i / S::kPieces;
            dma16_lanes(one(p.pages.k, ids, k, row) + 16 * (i % S::kPieces ^ swizzle(row)),
                        kt_at + 1024 * c);
        }
    };

    // V in registers: KiB r in row order.
    u4 vr[NR];
    const auto v_whole = [&](const size_t (&from)[KB]) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int row = STEP * (r / PERIOD), i = r % PERIOD;
            const unsigned at = row_of[i] * ROW + 16 * piece_of[i];
            vr[r] = *(const u4*)(p.pages.v + (from[row / 16] + row % 16 * ROW) + at);
        }
    };
    const auto v_any = [&](int ids, int k) {
        const int me = hidden_lane();
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int i = r % PERIOD * 64 + me;
            vr[r] = *(const u4*)(one(p.pages.v, ids, k, STEP * (r / PERIOD) + i / S::kPieces) +
                                 i % S::kPieces * 16);
        }
    };

    // The product of the weights w with the V in registers; also(i) amid its steps.
    char* const vt = kt + S::kKTile;
    u4 w[RB];
    const auto product = [&](auto also) {
#pragma unroll
        for (int r = 0; r < NR; ++r)
            *(u4*)(vt + (STEP * (r / PERIOD) + row_of[r % PERIOD]) * S::kVRow +
                   16 * piece_of[r % PERIOD]) = vr[r];
        const char* from = vt + (4 * g + j / 4) * S::kVRow + j % 4 * 8;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            also(i);
            const u4 v = transposed(from + 32 * i, from + 32 * i + 16 * S::kVRow);
#pragma unroll
            for (int b = 0; b < RB; ++b) o[b][i] = mfma32<T>(v, w[b], o[b][i]);
        }
    };
    const auto meet = [&](int i) {
        if (i == NB / 2) lds_barrier();
    };

    if (k0 < k1) {
        // Pages of this tile (`ids`) and the next (`ids1`), and where whole tiles of the
        // two begin: K of the next tile and, a step later, its V lie alike.
        int ids = find(k0), ids1 = find(k0 + KT);
        size_t at[KB] = {}, at1[KB] = {};
        k_any(ids, k0);
        wait_vmcnt<0>();
        bool first = true, partial = false;
        for (int k = k0, turn = 0; k < k1; k += KT, turn ^= 1) {
            const bool more = k + KT < k1, whole = runs && k + KT <= k1;
            const bool whole1 = more && runs && k + 2 * KT <= k1;
            if (whole1) halves(ids1, k + KT, at1);
            f4 sc[RB][KB];
#pragma unroll
            for (int r = 0; r < NQ; ++r)
#pragma unroll
                for (int h = 0; h < KB; ++h) {
                    const u4 a = *(const u4*)(kt + (16 * h + j) * S::kRow +
                                              16 * (4 * r + g ^ swizzle(j)));
#pragma unroll
                    for (int b = 0; b < RB; ++b)
                        sc[b][h] = mfma32<T>(a, qr[b][r], r ? sc[b][h] : f4{0, 0, 0, 0});
                }
            char* const share =
                lds + kWaves * S::kWaveLds + turn * kWaves * S::kShare + lane * 16;
#pragma unroll
            for (int i = 0; i < RB * KB; ++i)
                *(f4*)(share + wave * S::kShare + i * kWave * 16) = sc[i / KB][i % KB];
            if (!first && partial)
#pragma unroll
                for (int r = 0; r < NR; ++r) odd |= clear_not_finite<T>(vr[r]);
            if (more) wait_lds();  // this K has been read
            if (!first && whole1) {
                product([&](int i) {
                    k_whole(at1, i);
                    meet(i);
                });
            } else {
                if (more) k_any(ids1, k + KT);
                if (first)
                    meet(NB / 2);
                else
                    product(meet);
            }
            const int after = find(k + 2 * KT);
            if (!first && whole)
                v_whole(at);
            else
                v_any(ids, k);
            ids = ids1;
            ids1 = after;
#pragma unroll
            for (int i = 0; i < RB * KB; ++i) {
                f4 sum = *(f4*)(share + i * kWave * 16);
#pragma unroll
                for (int u = 1; u < kWaves; ++u)
                    sum += *(f4*)(share + u * S::kShare + i * kWave * 16);
                sc[i / KB][i % KB] = sum;
            }
            partial = k + KT > least;  // some row does not see all of the tile
            float keep[RB];
            if (weights(p, sc, partial, k + 4 * g, seen, m, l, keep))
#pragma unroll
                for (int b = 0; b < RB; ++b)
#pragma unroll
                    for (int i = 0; i < NB; ++i) o[b][i] *= keep[b];
#pragma unroll
            for (int b = 0; b < RB; ++b) w[b] = pack8<T>(sc[b][0], sc[b][1]);
            first = false;
#pragma unroll
            for (int h = 0; h < KB; ++h) at[h] = at1[h];
            // The next K has arrived: it was asked for before the NR loads of this V.
            if (more) wait_vmcnt<NR>();
        }
        if (partial)
#pragma unroll
            for (int r = 0; r < NR; ++r) odd |= clear_not_finite<T>(vr[r]);
        product([](int) {});
    }
    if (__ballot(odd))
        for (int c = max(k0, least / KT * KT); c < k1; ++c)
            if (const char* v = it.row_of_v(p, c, ROW))
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    const f4 x = odd_values<T>(v + (col0 + 16 * i + 4 * g) * 2);
#pragma unroll
                    for (int b = 0; b < RB; ++b)
                        if (c < seen[b]) o[b][i] += x;
                }
    const bool none = __ballot(bad) != 0;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const float sum = none ? NAN : wave_sum16_groups(l[b]);
        const int row = kRows * b + j;
        if (row < it.rows)
#pragma unroll
            for (int i = 0; i < NB; ++i)
                store<T, kDim, PREFIX>(p, it, row, col0 + 16 * i + 4 * g, o[b][i], m[b] * p.c2,
                                       sum);
    }
}

}  // namespace cache
}  // namespace xattn
