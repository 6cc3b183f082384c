// Cache attention in 16 bits, heads of up to 256, many rows (tile_item): prompts,
// and a shared prefix under the rows of a whole batch.  The matrix operands are
// those of xattn_cache_few.h.
//
// Each of the four wavefronts holds RB blocks of sixteen rows; all share tiles of K
// and V in LDS, so an operand read from LDS feeds RB matrix instructions.  There are
// two of each tile: DMA fills one pair, piece by piece between the matrix
// instructions, while the other is worked on; one barrier a tile.  Two workgroups
// share a CU (three at 64), and the wavefronts at their scores go before those at
// their softmax (s_setprio: 151 us in the case below, 163 without, 158 for the product
// with V as well).  Weights are taken relative to a maximum that is renewed only when a
// score exceeds it by kLag (in exponents of 2), so that the output is rarely rescaled;
// they stay below 2^kLag, far from the range of either type.
//
// Bound by the issue of matrix and vector instructions, which fill 45 % and 54 % of a
// SIMD's cycles in a causal prompt of 4,096 tokens, 32 heads on 8 kv heads of 128:
// 147 us, 935 TFLOP/s of what the mask leaves (a large matrix product: 1,167).  At 64
// half the matrix instructions meet the same number of weights: eight sequences of
// 2,048 tokens over 4,096 keys run at 695, at 128 at 872.
#pragma once

#include "xattn_cache_item.h"

namespace xattn {
namespace cache {

template <int D>
struct TileShape {
    static constexpr int kBlocks = D > 128 ? 1 : 2;       // row blocks of a wavefront (RB)
    static constexpr int kRows = 16 * kBlocks * kWaves;   // rows of a workgroup
    static constexpr int kKeys = D > 128 ? 32 : 64;       // keys of a tile
    static constexpr int kPieces = D / 8;                 // 16-byte pieces of a row
    static constexpr int kLoads = kKeys * kPieces / 256;  // pieces of a thread, of K and of V
    static constexpr int kTile = kKeys * D * 2;           // bytes of a tile in LDS
    static constexpr int kLds = 4 * kTile;
    // What a row's piece numbers are xored with in LDS: rows 0 .. 7 put a column's
    // 32 bytes into eight different eighths of the banks.
    static __device__ int swizzle(int row) { return D == 64 ? row / 2 % 4 * 2 : row % 8 * 2; }
};

template <typename T, int D, bool PREFIX>
__device__ __forceinline__ void tile_item(const AttendParams& p, unsigned block, char* lds) {
    typedef TileShape<D> S;
    constexpr int RB = S::kBlocks, KT = S::kKeys, KB = KT / 16, NL = S::kLoads;
    constexpr int DS = D / 32, DB = D / 16, LR = D * 2;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int j = lane % 16, g = lane / 16;
    Item it;
    if (!find_item<S::kRows, PREFIX>(p, block, &it)) return;
    const Sequence& s = it.s;
    const int k0 = it.k0, k1 = it.k1;

    int seen[RB];
    u4 q[RB][DS];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const Row r = it.row(p, min(16 * (wave * RB + b) + j, it.rows - 1));
        seen[b] = min(s.seen(r.token, it.causal), k1);
        const T* from = (const T*)p.q + r.token * p.qs + (long long)r.head * D + 8 * g;
#pragma unroll
        for (int i = 0; i < DS; ++i) q[b][i] = *(const u4*)(from + 32 * i) ^ p.sign;
    }
    f4 o[RB][DB], l[RB];  // l: the sum of a row's weights, four times
    float m[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        m[b] = -INFINITY;
        l[b] = f4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < DB; ++i) o[b][i] = f4{0, 0, 0, 0};
    }

    // A wavefront's pieces of a tile: AT_ONCE rows to a DMA of 1 KiB, the workgroup
    // STRIDE.  A row's pieces are permuted in LDS by swizzle(row): with rows whose
    // bytes are a power of two, eight rows of one column would share their banks,
    // and DMA leaves no room for padding.  Where AT_ONCE divides the page size its
    // rows lie on one page, and their address is one scalar plus a lane's constant
    // offset; a lane's own address otherwise, and where rows behind the last key
    // repeat it.
    constexpr int AT_ONCE = 64 / S::kPieces, STRIDE = kWaves * AT_ONCE;
    const int wave_row = __builtin_amdgcn_readfirstlane(wave * AT_ONCE);
    const int lane_row = lane / S::kPieces;
    const unsigned lane_byte =
        16u * (lane % S::kPieces ^ S::swizzle(wave * AT_ONCE + lane_row));
    const bool runs = p.pages.page_size.d % AT_ONCE == 0;
    const unsigned size = p.pages.page_size.d;
    bool bad = false, odd = false;
    int ids;  // lane's page of the next tile: that of its key lane % KT
    const auto find = [&](int k) {
        ids = it.table[p.pages.page_size.div((unsigned)min(k + lane % KT, k1 - 1))];
    };
    DmaSrc k_pool, v_pool;
    dma_base2(p.pages.k, p.pages.v, k_pool, v_pool);
    const unsigned lds0 = lds_u32(lds);
    // A tile's i-th pieces of K and V.  Whole tiles of pages as above: their
    // sources and the destination are prepared together, then asked for.
    struct Piece1 {
        DmaSrc k, v;
        unsigned to;
    };
    const unsigned from = lane_row * (D * 2) + lane_byte;
    const auto piece = [&](int t, int k, int i) {
        const int at_row = STRIDE * i + wave_row;
        const unsigned key = (unsigned)(k + at_row);
        const int page = __builtin_amdgcn_readlane(ids, at_row);
        const bool ok = page >= 0 && (unsigned)page < p.pages.num_pages;
        bad |= !ok;
        const unsigned row = ((ok ? (unsigned)page : 0u) * p.pages.kv_heads + it.kv_head) * size +
                             (key - p.pages.page_size.div(key) * size);
        const size_t at = (size_t)row * (D * 2);
        return Piece1{k_pool + at, v_pool + at,
                      lds0 + (t & 1) * 2 * S::kTile + at_row * (D * 2)};
    };
    const auto load_any = [&](int t, int k) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int at_row = STRIDE * i + wave_row;
            const unsigned to = lds0 + (t & 1) * 2 * S::kTile + at_row * (D * 2);
            const unsigned key = (unsigned)min(k + at_row + lane_row, k1 - 1);
            const int page = __shfl(ids, at_row + lane_row);
            const bool ok = page >= 0 && (unsigned)page < p.pages.num_pages;
            bad |= !ok;
            const unsigned row = ((ok ? (unsigned)page : 0u) * p.pages.kv_heads + it.kv_head) *
                                     size + (key - p.pages.page_size.div(key) * size);
            const size_t at = (size_t)row * (D * 2) + lane_byte;
            dma16_lanes(p.pages.k + at, to);
            dma16_lanes(p.pages.v + at, to + S::kTile);
        }
    };
    // The tile loaded last has arrived for this wavefront; infinities and NaN in
    // its pieces of V are cleared if some rows do not see all of the tile.
    const auto arrived = [&](int t, int k) {
        wait_vmcnt<0>();
        if (k + KT > it.least)
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                u4* at = (u4*)(lds + ((t & 1) * 2 + 1) * S::kTile +
                               (wave_row + i * STRIDE) * (D * 2) + lane * 16);
                u4 x = *at;
                if (clear_not_finite<T>(x)) {
                    odd = true;
                    *at = x;
                }
            }
    };

    if (k0 < k1) {
        find(k0);
        load_any(0, k0);
        find(k0 + KT);
        arrived(0, k0);
    }
    lds_barrier();
    int t = 0;
    for (int k = k0; k < k1; k += KT, ++t) {
        const bool more = k + KT < k1;
        const char* kt = lds + (t & 1) * 2 * S::kTile;
        const char* vt = kt + S::kTile;
        f4 sc[RB][KB];
        u4 a[2][DS];
        const auto read_k = [&](int h) {
#pragma unroll
            for (int i = 0; i < DS; ++i)
                a[h & 1][i] =
                    *(const u4*)(kt + (16 * h + j) * LR + 16 * (4 * i + g ^ S::swizzle(j)));
        };
        const auto scores = [&](int h, int from, int to) {
#pragma unroll
            for (int i = from; i < to; ++i)
#pragma unroll
                for (int b = 0; b < RB; ++b)
                    sc[b][h] = mfma32<T>(a[h & 1][i], q[b][i], i ? sc[b][h] : f4{0, 0, 0, 0});
        };
        __builtin_amdgcn_s_setprio(1);
        read_k(0);
        if (runs && k + 2 * KT <= k1) {
            // The next tile is asked for piece by piece between the products (the
            // path to memory takes a wavefront's requests no faster), each read of
            // LDS before the requests that it need not wait for.
#pragma unroll
            for (int h = 0; h < KB; ++h) {
                if (h + 1 < KB) read_k(h + 1);
#pragma unroll
                for (int i = h * NL / KB; i < (h + 1) * NL / KB; ++i) {
                    const Piece1 x = piece(t + 1, k + KT, i);
                    dma16_m0<0>(x.k, from, x.to);
                    dma16_m0<0>(x.v, from, x.to + S::kTile);
                }
                scores(h, 0, DS);
            }
        } else {
            if (more) load_any(t + 1, k + KT);
#pragma unroll
            for (int h = 0; h < KB; ++h) {
                if (h + 1 < KB) read_k(h + 1);
                scores(h, 0, DS);
            }
        }
        if (more) find(k + 2 * KT);
        __builtin_amdgcn_s_setprio(0);
        const bool partial = k + KT > it.least;
        if (partial) {
            int key = k + 4 * g;
            asm volatile("" : "+v"(key));  // keeps the comparisons in this branch
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int h = 0; h < KB; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (key + 16 * h + i >= seen[b]) sc[b][h][i] = -INFINITY;
        }
        float top[RB];
        bool past = false;
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            top[b] = -INFINITY;
#pragma unroll
            for (int h = 0; h < KB; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) top[b] = fmaxf(top[b], sc[b][h][i]);
            top[b] = wave_max16_groups(top[b]);
            past |= top[b] > m[b] + p.lag;
        }
        if (__ballot(past))
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                const float to = fmaxf(m[b], top[b]);
                const float keep = to == -INFINITY ? 1.0f : fast_exp2((m[b] - to) * p.c2);
                l[b] *= keep;
#pragma unroll
                for (int i = 0; i < DB; ++i) o[b][i] *= keep;
                m[b] = to;
            }
        u4 w[RB][KB / 2];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const float ref = m[b] == -INFINITY ? 0.0f : m[b] * p.c2;
#pragma unroll
            for (int h = 0; h < KB; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sc[b][h][i] = fast_exp2(__builtin_fmaf(sc[b][h][i], p.c2, -ref));
#pragma unroll
            for (int h = 0; h < KB / 2; ++h) {
                w[b][h] = u4{pack2<T>(sc[b][2 * h][0], sc[b][2 * h][1]),
                             pack2<T>(sc[b][2 * h][2], sc[b][2 * h][3]),
                             pack2<T>(sc[b][2 * h + 1][0], sc[b][2 * h + 1][1]),
                             pack2<T>(sc[b][2 * h + 1][2], sc[b][2 * h + 1][3])};
                l[b] = mfma32<T>(ones<T>(), w[b][h], l[b]);
            }
        }
        const int row = 4 * g + j / 4;  // of this lane's pieces of V
#pragma unroll
        for (int i = 0; i < DB; ++i) {
            const char* from =
                vt + row * LR + 16 * (2 * i + j % 4 / 2 ^ S::swizzle(row)) + j % 2 * 8;
#pragma unroll
            for (int h = 0; h < KB / 2; ++h) {
                const u4 a = transposed(from + 32 * h * LR, from + (32 * h + 16) * LR);
#pragma unroll
                for (int b = 0; b < RB; ++b) o[b][i] = mfma32<T>(a, w[b][h], o[b][i]);
            }
        }
        if (more) arrived(t + 1, k + KT);
        lds_barrier();
    }
    if (__syncthreads_or(bad))
#pragma unroll
        for (int b = 0; b < RB; ++b) l[b][0] = NAN;
    if (__syncthreads_or(odd))
        for (int k = max(k0, it.least / KT * KT); k < k1; ++k)
            if (const char* v = it.row_of_v(p, k, D * 2))
#pragma unroll
                for (int i = 0; i < DB; ++i) {
                    const f4 x = odd_values<T>(v + (16 * i + 4 * g) * 2);
#pragma unroll
                    for (int b = 0; b < RB; ++b)
                        if (k < seen[b]) o[b][i] += x;
                }
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const int row = 16 * (wave * RB + b) + j;
        if (row < it.rows)
#pragma unroll
            for (int i = 0; i < DB; ++i)
                store<T, D, PREFIX>(p, it, row, 16 * i + 4 * g, o[b][i], m[b] * p.c2, l[b][0]);
    }
}

}  // namespace cache
}  // namespace xattn
