// Cache attention in 32 bits, and in 16 bits at dim 768 (ring_item): sixteen rows.
//
// The scores and weights lie in the lanes as in xattn_cache_few.h (16x16x4 MFMAs in
// 32 bits: tiles of 16 keys, a weight's register is its operand's).  Up to dim 256
// every wavefront has tiles of its own; at 768 the four share theirs and own 192
// columns each, of Q, K, V and the output, and sum their shares of the scores
// through LDS.
//
// K arrives by DMA in a slice of LDS of the wavefront's own.  Straight into the
// operand's layout, whose neighbouring lanes are different rows, a KiB would hold
// the CU's path to memory for 64 cycles instead of 16, which bounded this form at
// 3.7 us a tile of 768 columns where the matrix instructions take 1.3.  Its pieces
// are swizzled so that neighbouring rows use distinct banks.  V comes in whole rows
// into registers: in 32 bits a lane's 16 bytes are one element each of four matrix
// operands, whose columns are dealt accordingly (column 64 (b / 4) + 4 r + b % 4 is
// row r of block b); in 16 bits they pass through LDS to be read transposed.
//
// A tile's scores come before the product of the tile before it with V, under which
// the shares of the scores are exchanged; its softmax comes last.  What the next
// steps need is asked for piece by piece between the matrix instructions (in one
// run it would hold the wavefront until the path to memory has taken it, 968 cycles
// for V at 768 columns in 32 bits): in 32 bits the next K under the scores, into the
// other of two slots, and this tile's V under the product, register by register as
// the old ones have been used; in 16 bits, whose LDS has room for one K only, the
// next K under the product and V behind it.
#pragma once

#include "xattn_cache_item.h"

namespace xattn {
namespace cache {

template <typename T, int D>
struct RingShape {
    static constexpr bool kWide = sizeof(T) == 4;
    static constexpr int kCols = D > 256 ? kWaves : 1;  // wavefronts that share a tile
    static constexpr int kDW = D / kCols;               // columns of a wavefront
    static constexpr int kKeys = kWide ? 16 : 32;       // keys of a tile
    static constexpr int kRegs = kDW / 16;              // KiB of a wavefront's K, or V, in a tile
    static constexpr int kBlocks = kDW / 16;            // 16-column blocks of the output
    static constexpr int kRow = kDW * (int)sizeof(T);   // bytes of a row's columns
    static constexpr int kPieces = kRow / 16;
    // A KiB holds 64 pieces of consecutive rows; kPeriod KiB hold kStep whole rows.
    static constexpr int kPeriod =
        64 % kPieces == 0 ? 1 : kPieces % 16 == 0 ? kPieces / 16 : kPieces / 8;
    static constexpr int kStep = 64 * kPeriod / kPieces;
    static constexpr int kKTile = kRegs * 1024;
    static constexpr int kSlots = kWide ? 2 : 1;        // K tiles of a wavefront in LDS
    static constexpr int kVRow = kRow + 32;             // in LDS; 32 bytes of padding deal four
                                                        // rows to distinct banks
    static constexpr int kVTile = kWide ? 0 : kKeys * kVRow;
    static constexpr int kORow = kDW + 4;               // floats of an output row in LDS
    static constexpr int kOut = kCols > 1 ? 0 : kRows * kORow * 4;
    static constexpr int kTiles = kSlots * kKTile + kVTile;
    static constexpr int kWaveLds = kTiles > kOut ? kTiles : kOut;
    static constexpr int kShare = kKeys * kRows * 4;    // bytes of a wavefront's share of scores
    static constexpr int kShares = kCols > 1 ? 2 * kWaves * kShare : 0;
    static constexpr int kStats = kWaves * kRows * 8;   // maxima and sums
    static constexpr int kLds = kWaves * kWaveLds + kShares + kStats;
    // What a row's piece numbers in LDS are xored with: eight rows put a column's
    // 32 bytes into eight different eighths of the banks.
    static constexpr __device__ int swizzle(int row) {
        return kRow % 256 == 0 ? row % 8 * 2 : row / 2 % 4 * 2;
    }
};

template <typename T, int D, bool PREFIX>
__device__ __forceinline__ void ring_item(const AttendParams& p, unsigned block, char* lds) {
    typedef RingShape<T, D> S;
    constexpr int KT = S::kKeys, KB = KT / 16, NR = S::kRegs, NB = S::kBlocks;
    constexpr bool WIDE = S::kWide, SHARED = S::kCols > 1;
    constexpr int PERIOD = S::kPeriod, STEP = S::kStep, SIZE = (int)sizeof(T), ROW = D * SIZE;
    float2(*const stats)[kRows] = (float2(*)[kRows])(lds + S::kLds - S::kStats);
    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int j = lane % 16, g = lane / 16;

    Item it;
    if (!find_item<kRows, PREFIX>(p, block, &it)) return;
    const Sequence& s = it.s;
    const int least = it.least, k0 = it.k0, k1 = it.k1;
    const Row mine = it.row(p, min(j, it.rows - 1));
    const int seen = min(s.seen(mine.token, it.causal), k1);

    // Q: register r holds elements 16 r + 4 g on (32 bits), 32 r + 8 g on (16 bits).
    constexpr int NQ = WIDE ? NR : NR / 2;
    const int col0 = SHARED ? wave * S::kDW : 0;
    u4 qr[NQ];
    {
        const char* q = (const char*)((const T*)p.q + mine.token * p.qs +
                                      (long long)mine.head * D + col0) + 16 * g;
#pragma unroll
        for (int r = 0; r < NQ; ++r) qr[r] = *(const u4*)(q + 64 * r) ^ p.sign;
    }
    f4 o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = f4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;
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
    const auto half = [&](const char* pool, int ids, int k, int h) {  // rows 16 h on
        const unsigned row = row_at(__builtin_amdgcn_readlane(ids, 16 * h), k + 16 * h);
        return pool + (size_t)row * ROW + col0 * SIZE;
    };
    const auto one = [&](const char* pool, int ids, int k, int r) {  // row r
        const unsigned row = row_at(__shfl(ids, r), (unsigned)min(k + r, k1 - 1));
        return pool + (size_t)row * ROW + col0 * SIZE;
    };

    // K by DMA: KiB c of a tile.
    char* const kt = lds + wave * S::kWaveLds;
    const unsigned kt_at = __builtin_amdgcn_readfirstlane(lds_u32(kt));
    int k_row[PERIOD], k_piece[PERIOD];
#pragma unroll
    for (int i = 0; i < PERIOD; ++i) {
        k_row[i] = (i * 64 + lane) / S::kPieces;
        k_piece[i] = (i * 64 + lane) % S::kPieces;
    }
    const auto k_from = [&](int c) {  // lane's piece of its row's columns, in bytes
        const int row = STEP * (c / PERIOD) + k_row[c % PERIOD];
        return 16 * (k_piece[c % PERIOD] ^ S::swizzle(row));
    };
    const auto dma_whole = [&](const DmaSrc (&from)[KB], int slot, int c) {
        const int row = STEP * (c / PERIOD);
        dma16_m0<0>(from[row / 16] + (size_t)(row % 16 * ROW),
                    (unsigned)(k_row[c % PERIOD] * ROW + k_from(c)),
                    kt_at + slot * S::kKTile + 1024 * c);
    };
    DmaSrc pool;
    {
        DmaSrc same;
        dma_base2(p.pages.k, p.pages.k, pool, same);
    }
    const auto k_whole = [&](int ids, int k, DmaSrc (&from)[KB]) {
#pragma unroll
        for (int h = 0; h < KB; ++h)
            from[h] = pool + (size_t)(half(p.pages.k, ids, k, h) - p.pages.k);
    };
    const auto dma_any = [&](int ids, int k, int slot) {
#pragma unroll
        for (int c = 0; c < NR; ++c)
            dma16_lanes(one(p.pages.k, ids, k, STEP * (c / PERIOD) + k_row[c % PERIOD]) + k_from(c),
                        kt_at + slot * S::kKTile + 1024 * c);
    };

    // V in registers.  32 bits: register r is columns 64 (r / 4) + 4 j on of row 4 g +
    // r % 4.  16 bits: KiB r in row order.
    u4 vr[NR];
    const auto v_whole = [&](int ids, int k, const char* (&from)[KB]) {
#pragma unroll
        for (int h = 0; h < KB; ++h) from[h] = half(p.pages.v, ids, k, h);
    };
    const auto load_whole = [&](const char* const (&from)[KB], int r) {
        if constexpr (WIDE) {
            const unsigned at = 4 * g * ROW + 16 * j;
            vr[r] = *(const u4*)(from[0] + (r % 4 * ROW + 256 * (r / 4)) + at);
        } else {
            const int row = STEP * (r / PERIOD);
            const unsigned at = k_row[r % PERIOD] * ROW + 16 * k_piece[r % PERIOD];
            vr[r] = *(const u4*)(from[row / 16] + row % 16 * ROW + at);
        }
    };
    const auto load_any = [&](int ids, int k) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            if constexpr (WIDE)
                vr[r] = *(const u4*)(one(p.pages.v, ids, k, 4 * g + r % 4) + 256 * (r / 4) + 16 * j);
            else
                vr[r] = *(const u4*)(one(p.pages.v, ids, k,
                                         STEP * (r / PERIOD) + k_row[r % PERIOD]) +
                                     16 * k_piece[r % PERIOD]);
        }
    };

    // The product of the weights `w` with the V in registers.  Between its steps comes
    // also(r); in 32 bits V's register r is free by then.
    char* const vt = kt + S::kSlots * S::kKTile;
    f4 w[KB];
    const auto product = [&](auto also) {
        if constexpr (WIDE) {
#pragma unroll
            for (int r = 0; r < NR; ++r) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    o[r / 4 * 4 + e] =
                        mfma4(__uint_as_float(vr[r][e]), w[0][r % 4], o[r / 4 * 4 + e]);
                also(r);
            }
        } else {
#pragma unroll
            for (int r = 0; r < NR; ++r)
                *(u4*)(vt + (STEP * (r / PERIOD) + k_row[r % PERIOD]) * S::kVRow +
                       16 * k_piece[r % PERIOD]) = vr[r];
            const u4 x = {pack2<T>(w[0][0], w[0][1]), pack2<T>(w[0][2], w[0][3]),
                          pack2<T>(w[KB - 1][0], w[KB - 1][1]), pack2<T>(w[KB - 1][2], w[KB - 1][3])};
            const char* from = vt + (4 * g + j / 4) * S::kVRow + j % 4 * 8;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                also(b);
                o[b] = mfma32<T>(transposed(from + 32 * b, from + 32 * b + 16 * S::kVRow), x, o[b]);
            }
        }
    };

    const int step = SHARED ? KT : kWaves * KT;
    int k = k0 + (SHARED ? 0 : wave * KT);
    if (k < k1) {
        int ids = find(k), ids1 = find(k + step);
        dma_any(ids, k, 0);
        wait_vmcnt<0>();
        bool first = true, partial = false;
        for (int turn = 0; k < k1; k += step, turn ^= 1) {
            const bool more = k + step < k1, whole = runs && k + KT <= k1;
            const bool whole1 = more && runs && k + step + KT <= k1;
            const int ids2 = find(k + 2 * step);
            f4 sc[KB];
            if constexpr (WIDE) {
                // in four sums, as a product takes longer to come out than to start
                const char* const from = kt + turn * S::kKTile + j * S::kRow;
                const auto scores = [&](auto also) {
                    f4 part[4];
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        const u4 a = *(const u4*)(from + 16 * (4 * r + g ^ S::swizzle(j)));
                        also(r);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            part[e] = mfma4(__uint_as_float(a[e]), __uint_as_float(qr[r][e]),
                                            r ? part[e] : f4{0, 0, 0, 0});
                    }
                    sc[0] = (part[0] + part[1]) + (part[2] + part[3]);
                };
                if (whole1) {
                    DmaSrc next[KB];
                    k_whole(ids1, k + step, next);
                    scores([&](int r) { dma_whole(next, turn ^ 1, r); });
                } else {
                    if (more) dma_any(ids1, k + step, turn ^ 1);
                    scores([](int) {});
                }
            } else {
#pragma unroll
                for (int r = 0; r < NQ; ++r)
#pragma unroll
                    for (int h = 0; h < KB; ++h) {
                        const u4 a = *(const u4*)(kt + (16 * h + j) * S::kRow +
                                                  16 * (4 * r + g ^ S::swizzle(j)));
                        sc[h] = mfma32<T>(a, qr[r], r ? sc[h] : f4{0, 0, 0, 0});
                    }
            }
            char* const share = lds + kWaves * S::kWaveLds + turn * kWaves * S::kShare;
            if constexpr (SHARED)
#pragma unroll
                for (int h = 0; h < KB; ++h)
                    *(f4*)(share + wave * S::kShare + (h * kWave + lane) * 16) = sc[h];
            // The product of the tile before.
            if (!first && partial)
#pragma unroll
                for (int r = 0; r < NR; ++r) odd |= clear_not_finite<T>(vr[r]);
            const auto meet = [&](int r) {
                if constexpr (SHARED)
                    if (r == NR / 2) lds_barrier();
            };
            if constexpr (WIDE) {
                if (!first && whole) {
                    const char* from[KB];
                    v_whole(ids, k, from);
                    product([&](int r) {
                        load_whole(from, r);
                        meet(r);
                    });
                } else {
                    if (first)
                        meet(NR / 2);
                    else
                        product(meet);
                    load_any(ids, k);
                }
            } else {
                if (more) wait_lds();  // this K has been read
                if (!first && whole1) {
                    DmaSrc next[KB];
                    k_whole(ids1, k + step, next);
                    product([&](int r) {
                        dma_whole(next, 0, r);
                        meet(r);
                    });
                } else {
                    if (more) dma_any(ids1, k + step, 0);
                    if (first)
                        meet(NR / 2);
                    else
                        product(meet);
                }
                if (whole) {
                    const char* from[KB];
                    v_whole(ids, k, from);
#pragma unroll
                    for (int r = 0; r < NR; ++r) load_whole(from, r);
                } else {
                    load_any(ids, k);
                }
            }
            if constexpr (SHARED)
#pragma unroll
                for (int h = 0; h < KB; ++h) {
                    sc[h] = *(f4*)(share + (h * kWave + lane) * 16);
#pragma unroll
                    for (int i = 1; i < kWaves; ++i)
                        sc[h] += *(f4*)(share + i * S::kShare + (h * kWave + lane) * 16);
                }
            partial = k + KT > least;  // some row does not see all of the tile
            const float keep = weights(p, sc, partial, k + 4 * g, seen, &m, &l);
            if (__ballot(keep != 1.0f))
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] *= keep;
#pragma unroll
            for (int h = 0; h < KB; ++h) w[h] = sc[h];
            first = false;
            ids = ids1;
            ids1 = ids2;
            // The next K has arrived: it was asked for before the NR loads of this V.
            if (more) wait_vmcnt<NR>();
        }
        if (partial)
#pragma unroll
            for (int r = 0; r < NR; ++r) odd |= clear_not_finite<T>(vr[r]);
        product([](int) {});
    }
    if (__ballot(odd))
        for (int t = k0 + (SHARED ? 0 : wave * KT); t < k1; t += step)
            for (int c = t; t + KT > least && c < min(t + KT, k1); ++c)
                if (const char* v = it.row_of_v(p, c, ROW))
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        f4 x;
                        if constexpr (WIDE) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float f = *(const float*)(
                                    v + (col0 + 64 * (b / 4) + 16 * g + 4 * i + b % 4) * 4);
                                x[i] = __builtin_isfinite(f) ? 0.0f : f;
                            }
                        } else {
                            x = odd_values<T>(v + (col0 + 16 * b + 4 * g) * 2);
                        }
                        if (c < seen) o[b] += x;
                    }
    l = wave_sum16_groups(l);
    if (__ballot(bad)) l = NAN;

    // In 32 bits four blocks hold four neighbouring columns each.
    const auto quads = [&](auto put) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if constexpr (WIDE) {
                if (b % 4 == 0)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        put(16 * b + 16 * g + 4 * i,
                            f4{o[b][i], o[b + 1][i], o[b + 2][i], o[b + 3][i]});
            } else {
                put(16 * b + 4 * g, o[b]);
            }
        }
    };
    if constexpr (SHARED) {
        if (j < it.rows)
            quads([&](int col, f4 x) {
                store<T, D, PREFIX>(p, it, j, col0 + col, x, m * p.c2, l);
            });
    } else {
        if (lane < kRows) stats[wave][lane] = {m * p.c2, l};
        float* part = (float*)kt + j * S::kORow;
        quads([&](int col, f4 x) { *(f4*)(part + col) = x; });
        __syncthreads();
        join_and_store<T, D, PREFIX>(p, it, stats, lds, S::kWaveLds, S::kORow);
    }
}

}  // namespace cache
}  // namespace xattn
