// Cache attention in 32 bits (wide_item): RB blocks of sixteen rows, one or two.
//
// Tiles of 16 keys on 16x16x4 MFMAs.  The scores and weights lie in the lanes as in
// xattn_cache_few.h; a weight's register is the operand of its key.  Up to dim 128
// every wavefront has tiles of its own; from 256 on the four share theirs and own a
// quarter of the columns each, of Q, K, V and the output, and sum their shares of the
// scores through LDS.
//
// Beside these MFMAs another wavefront's vector instructions do not issue, so the
// loop has to leave the matrix pipe as little as it can: K and V come by DMA into
// LDS of the wavefront's own, K into two slots, V into one, requested KiB by KiB
// between the matrix instructions (all at once they would hold the wavefront until
// the path to memory has taken them: 968 cycles for V at 768 columns), and what
// the wavefront waits for was asked for a whole tile before:
//
//   scores of tile t (K of tile t + 1 asked for)  ->  shares of the scores
//   product of tile t - 1 with V, its KiB replaced by those of tile t once read;
//     half way through it the shares of the scores are there
//   softmax of tile t
//
// K's pieces are swizzled in LDS so that neighbouring rows use distinct banks.  V's
// KiB r is what lane (j, g) needs at step r: columns 64 (r / 4) + 4 j .. + 3 of key
// 4 g + r % 4, one element each of four matrix operands; so row i of the output's block
// b is column 64 (b / 4) + 4 i + b % 4.
//
// The waits count the DMA by themselves, so no other load may stand between: the
// pages of 64 tiles are looked up at a time.
//
// Few rows are bound by memory (32 sequences of 4,000 keys, one token each: 5.2 to 5.6
// TB/s at all dims), many by the matrix instructions and what the wavefront does
// between them: 64 rows over 50,176 keys of 768 take 122 us with the matrix pipe busy
// for 57 % of them, 1,024 tokens over 1,500 keys run at 67 TFLOP/s at 64, 82 at 128, 68
// at 256 (a large matrix product: 153).
#pragma once

#include "xattn_cache_item.h"

namespace xattn {
namespace cache {

template <int D, int RB>
struct WideShape {
    static constexpr int kCols = D > 128 ? kWaves : 1;  // wavefronts that share a tile
    static constexpr int kDW = D / kCols;               // columns of a wavefront
    static constexpr int kKeys = 16;                    // keys of a tile
    static constexpr int kRegs = kDW / 16;              // KiB of a wavefront's K, or V, in a tile
    static constexpr int kRow = kDW * 4;                // bytes of a row's columns
    static constexpr int kPieces = kRow / 16;
    // A KiB of K holds 64 pieces of consecutive rows; kPeriod KiB hold kStep whole rows.
    static constexpr int kPeriod = 64 % kPieces == 0 ? 1 : kPieces / 16;
    static constexpr int kStep = 64 * kPeriod / kPieces;
    static constexpr int kTile = kRegs * 1024;
    static constexpr int kWaveLds = 3 * kTile;
    static constexpr int kORow = kDW + 4;               // floats of an output row in LDS
    static constexpr int kShare = RB * kKeys * kRows * 4;  // bytes of a wavefront's share of scores
    static constexpr int kShares = kCols > 1 ? 2 * kWaves * kShare : 0;
    static constexpr int kStats = kCols > 1 ? 0 : kWaves * RB * kRows * 8;  // maxima and sums
    static constexpr int kLds = kWaves * kWaveLds + kShares + kStats;
    static_assert(kCols > 1 || RB * kRows * kORow * 4 <= kWaveLds, "the output takes the tiles' room");
    static_assert(2 * kRegs < 64, "waits of up to 63 loads");
};

template <int D, int RB, bool PREFIX>
__device__ __forceinline__ void wide_item(const AttendParams& p, unsigned block, char* lds) {
    typedef WideShape<D, RB> S;
    constexpr int KT = S::kKeys, NR = S::kRegs, ROW = D * 4;
    constexpr int PERIOD = S::kPeriod, STEP = S::kStep;
    constexpr bool SHARED = S::kCols > 1;
    constexpr int AHEAD = RB > 1 ? 2 : 3;  // steps of 4 RB products that LDS is read ahead of use
    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int j = lane % 16, g = lane / 16;

    Item it;
    if (!find_item<RB * kRows, PREFIX>(p, block, &it)) return;
    const Sequence& s = it.s;
    const int least = it.least, k0 = it.k0, k1 = it.k1;

    // Q: register r of lane (j, g) holds elements 16 r + 4 g .. + 3 of row j.
    const int col0 = SHARED ? wave * S::kDW : 0;
    int seen[RB];
    u4 q[RB][NR];
    f4 o[RB][NR];
    float m[RB], l[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const Row mine = it.row(p, min(kRows * b + j, it.rows - 1));
        seen[b] = min(s.seen(mine.token, it.causal), k1);
        const float* from =
            (const float*)p.q + mine.token * p.qs + (long long)mine.head * D + col0 + 4 * g;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            q[b][r] = *(const u4*)(from + 16 * r) ^ p.sign;
            o[b][r] = f4{0, 0, 0, 0};
        }
        m[b] = -INFINITY;
        l[b] = 0.0f;
    }
    bool bad = false, odd = false;

    // Where tiles lie.  A tile is on one page where sixteen divides the page size: its
    // rows are then one scalar plus a lane's constant offset.  A lane's own address
    // otherwise, and where rows behind the last key repeat it.
    const unsigned size = p.pages.page_size.d;
    const bool runs = size % KT == 0;
    const int step = SHARED ? KT : kWaves * KT;
    const int start = k0 + (SHARED ? 0 : wave * KT);
    const auto row_at = [&](int page, unsigned key) {
        const bool ok = page >= 0 && (unsigned)page < p.pages.num_pages;
        bad |= !ok;
        return ((ok ? (unsigned)page : 0u) * p.pages.kv_heads + it.kv_head) * size +
               (key - p.pages.page_size.div(key) * size);
    };
    int ids = 0;  // lane i's: the page of tile i of 64
    const auto find = [&](int tile) {
        const long long key = start + (long long)(tile + lane) * step;
        ids = it.table[p.pages.page_size.div((unsigned)min(key, (long long)k1 - 1))];
    };
    const auto whole_at = [&](int tile) {  // byte offset of a whole tile: a scalar
        const unsigned row = row_at(__builtin_amdgcn_readlane(ids, tile % kWave),
                                    (unsigned)(start + tile * step));
        return (size_t)row * ROW + col0 * 4;
    };
    // (The lane read through an empty asm: what the rare path derives from it is
    // otherwise kept in registers across the loop.)
    const auto hidden_lane = [&]() {
        int i = lane;
        asm volatile("" : "+v"(i));
        return i;
    };
    const auto own_at = [&](const char* pool, int k, int row) {
        const unsigned key = (unsigned)min(k + row, k1 - 1);
        return pool + (size_t)row_at(it.table[p.pages.page_size.div(key)], key) * ROW + col0 * 4;
    };

    char* const kt = lds + wave * S::kWaveLds;
    const unsigned kt_at = __builtin_amdgcn_readfirstlane(lds_u32(kt));
    const unsigned vt_at = kt_at + 2 * S::kTile;
    const DmaSrc k_pool = dma_base(p.pages.k), v_pool = dma_base(p.pages.v);
    const auto swizzle = [](int row) { return row % 8 * 2; };
    const auto k_whole = [&](size_t at, int slot, int c) {  // KiB c of a tile of K
        const int i = c % PERIOD * 64 + lane, row = STEP * (c / PERIOD) + i / S::kPieces;
        dma16_m0<0>(k_pool + (at + (size_t)(STEP * (c / PERIOD) * ROW)),
                    (unsigned)(i / S::kPieces * ROW + 16 * (i % S::kPieces ^ swizzle(row))),
                    kt_at + slot * S::kTile + 1024 * c);
    };
    const auto v_whole = [&](size_t at, int r) {
        dma16_m0<0>(v_pool + (at + (size_t)(r % 4 * ROW + 256 * (r / 4))),
                    (unsigned)(4 * g * ROW + 16 * j), vt_at + 1024 * r);
    };
    const auto k_any = [&](int k, int slot) {
        const int me = hidden_lane();
        const char* from[NR];
#pragma unroll
        for (int c = 0; c < NR; ++c) {
            const int i = c % PERIOD * 64 + me, row = STEP * (c / PERIOD) + i / S::kPieces;
            from[c] = own_at(p.pages.k, k, row) + 16 * (i % S::kPieces ^ swizzle(row));
        }
#pragma unroll
        for (int c = 0; c < NR; ++c)
            dma16_lanes(from[c], kt_at + slot * S::kTile + 1024 * c);
    };
    const auto v_any = [&](int k) {
        const int me = hidden_lane();
        const char* from[4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
            from[r] = own_at(p.pages.v, k, me / 16 * 4 + r) + me % 16 * 16;
#pragma unroll
        for (int r = 0; r < NR; ++r)
            dma16_lanes(from[r % 4] + 256 * (r / 4), vt_at + 1024 * r);
    };

    unsigned k_lane[4];  // where lane (j, g) reads pieces 4 i + g of row j
#pragma unroll
    for (int i = 0; i < 4; ++i) k_lane[i] = kt_at + j * S::kRow + 16 * (4 * i + g ^ swizzle(j));

    // Scores of the tile in a slot; also(r) comes amid the products of step r.
    f4 sc[RB][1];
    const auto scores = [&](int slot, auto also) {
        // in several sums, as a product takes longer to come out than to start
        constexpr int SUMS = RB > 1 ? 2 : 4;
        // Four addresses, and constants: a vector instruction between the products
        // would wait until the matrix pipe has run empty.
        lds_char* from[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            unsigned at = k_lane[i] + slot * S::kTile;
            asm volatile("" : "+v"(at));
            from[i] = (lds_char*)(uintptr_t)at;
        }
        f4 part[RB][SUMS];
        u4 k4[AHEAD + 1];
        const auto read = [&](int r) {
            k4[r % (AHEAD + 1)] = *(const lds_u4*)(from[r % 4] + 256 * (r / 4));
        };
#pragma unroll
        for (int r = 0; r < AHEAD; ++r) read(r);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            if (r + AHEAD < NR) read(r + AHEAD);
            __builtin_amdgcn_sched_barrier(0);  // here: the reads would sink to their use
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
                for (int b = 0; b < RB; ++b)
                    part[b][e % SUMS] =
                        mfma4(__uint_as_float(k4[r % (AHEAD + 1)][e]), __uint_as_float(q[b][r][e]),
                              r || e >= SUMS ? part[b][e % SUMS] : f4{0, 0, 0, 0});
                if (e == 1) also(r);
            }
        }
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            sc[b][0] = part[b][0];
#pragma unroll
            for (int e = 1; e < SUMS; ++e) sc[b][0] += part[b][e];
        }
    };

    // The product of the weights w with the tile in V; before(r) comes before KiB r is
    // read, after(r) when it has been, amid its products.  `partial`: infinities and NaN are cleared.
    lds_char* const v_lane = (lds_char*)(uintptr_t)(vt_at + 16 * lane);
    f4 w[RB];
    const auto product = [&](bool partial, auto before, auto after) {
        u4 v4[AHEAD + 1];
        const auto read = [&](int r) {
            before(r);
            v4[r % (AHEAD + 1)] = *(const lds_u4*)(v_lane + 1024 * r);
        };
#pragma unroll
        for (int r = 0; r < AHEAD; ++r) read(r);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            if (r + AHEAD < NR) read(r + AHEAD);
            u4 v = v4[r % (AHEAD + 1)];
            if (partial) odd |= clear_not_finite<float>(v);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
                for (int b = 0; b < RB; ++b)
                    o[b][r / 4 * 4 + e] =
                        mfma4(__uint_as_float(v[e]), w[b][r % 4], o[b][r / 4 * 4 + e]);
                if (e == 1) {
                    __builtin_amdgcn_sched_barrier(0);  // KiB r has been read: it is in use
                    after(r);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    };
    const auto nothing = [](int) {};

    if (start < k1) {
        const int tiles = (k1 - start + step - 1) / step;
        const auto whole = [&](int t) { return runs && start + t * step + KT <= k1; };
        find(0);
        k_any(start, 0);
        wait_vmcnt<0>();
        size_t at = 0, at1 = 0;  // of this tile and the next, where they are whole
        bool partial = false;
        for (int t = 0; t < tiles; ++t) {
            const bool more = t + 1 < tiles, whole0 = t > 0 && whole(t);
            const bool whole1 = more && whole(t + 1);
            const int k = start + t * step;
            if (whole1) {
                if ((t + 1) % kWave == 0) {
                    find(t + 1);
                    wait_vmcnt<0>();
                }
                at1 = whole_at(t + 1);
                scores(t & 1, [&](int r) { k_whole(at1, t + 1 & 1, r); });
            } else {
                if (more) k_any(k + step, t + 1 & 1);
                scores(t & 1, nothing);
            }
            char* const share =
                lds + kWaves * S::kWaveLds + (t & 1) * kWaves * S::kShare + lane * 16;
            if constexpr (SHARED)
#pragma unroll
                for (int b = 0; b < RB; ++b)
                    *(f4*)(share + wave * S::kShare + b * kWave * 16) = sc[b][0];
            const auto meet = [&](int r) {
                if constexpr (SHARED)
                    if (r == NR / 2) lds_barrier();
            };
            if (whole0 && whole1 && !partial) {
                // The steady state.  Behind V's KiB r of the last tile, the NR - 1 - r others
                // were asked for, NR of the next K, and r - AHEAD or more of this V.
                product(false, [&](int r) { wait_vmcnt<2 * NR - 1 - AHEAD>(); },
                        [&](int r) {
                            v_whole(at, r);
                            meet(r);
                        });
            } else if (t > 0) {
                if (more)
                    wait_vmcnt<NR>();  // all but the next K
                else
                    wait_vmcnt<0>();
                product(partial, nothing, meet);
                wait_lds();  // this V has been read
                v_any(k);
            } else {
                meet(NR / 2);
                v_any(k);
            }
            if constexpr (SHARED)
#pragma unroll
                for (int b = 0; b < RB; ++b) {
                    f4 sum = *(f4*)(share + b * kWave * 16);
#pragma unroll
                    for (int i = 1; i < kWaves; ++i)
                        sum += *(f4*)(share + i * S::kShare + b * kWave * 16);
                    sc[b][0] = sum;
                }
            partial = k + KT > least;  // some row does not see all of the tile
            float keep[RB];
            if (weights(p, sc, partial, k + 4 * g, seen, m, l, keep))
#pragma unroll
                for (int b = 0; b < RB; ++b)
#pragma unroll
                    for (int i = 0; i < NR; ++i) o[b][i] *= keep[b];
#pragma unroll
            for (int b = 0; b < RB; ++b) w[b] = sc[b][0];
            at = at1;
            // The next K has arrived: the NR requests of this V came behind it.
            if (more) wait_vmcnt<NR>();
        }
        wait_vmcnt<0>();
        product(partial, nothing, nothing);
    }
    if (__ballot(odd))
        for (int t = start; t < k1; t += step)
            for (int c = t; t + KT > least && c < min(t + KT, k1); ++c)
                if (const char* v = it.row_of_v(p, c, ROW))
#pragma unroll
                    for (int i = 0; i < NR; ++i) {
                        f4 x;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float f = *(const float*)(
                                v + (col0 + 64 * (i / 4) + 16 * g + 4 * e + i % 4) * 4);
                            x[e] = __builtin_isfinite(f) ? 0.0f : f;
                        }
#pragma unroll
                        for (int b = 0; b < RB; ++b)
                            if (c < seen[b]) o[b][i] += x;
                    }

    const bool none = __ballot(bad) != 0;
    float2(*const stats)[RB * kRows] = (float2(*)[RB * kRows])(lds + S::kLds - S::kStats);
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const float sum = none ? NAN : wave_sum16_groups(l[b]);
        const int row = kRows * b + j;
        // four blocks hold four neighbouring columns each
#pragma unroll
        for (int i = 0; i < NR; i += 4)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = 16 * i + 16 * g + 4 * e;
                const f4 x = {o[b][i][e], o[b][i + 1][e], o[b][i + 2][e], o[b][i + 3][e]};
                if constexpr (SHARED) {
                    if (row < it.rows)
                        store<float, D, PREFIX>(p, it, row, col0 + col, x, m[b] * p.c2, sum);
                } else {
                    *(f4*)((float*)kt + row * S::kORow + col) = x;
                }
            }
        if constexpr (!SHARED)
            if (lane < kRows) stats[wave][row] = {m[b] * p.c2, sum};
    }
    if constexpr (!SHARED) {
        __syncthreads();
        join_and_store<float, D, PREFIX, RB * kRows>(p, it, stats, lds, S::kWaveLds, S::kORow);
    }
}

}  // namespace cache
}  // namespace xattn
