// Attention over a paged cache, with or without a prefix that the whole batch
// shares: o = sum_c e^(s_c - m) v_c / sum_c e^(s_c - m), s_c = scale q.k_c, in one
// pass over the keys with the running maximum m.
//
// The query heads of one kv head see the same keys, so a sequence's rows are
// its (token, head of the group) pairs, `group` to a token.  A work item is
// (kv head, sixteen rows, a range of keys) on one workgroup of four wavefronts;
// where there are fewer items than the device needs, the keys are divided and a
// second launch merges the parts.  For the prefix the rows are those of the whole
// batch, so that its keys are read once for sixteen rows of any sequences.
//
// cache_attend_kernel.  Scores are S^T = K Q^T on 16x16 MFMAs (keys on the M
// axis): lane (j = lane % 16, g = lane / 16) ends with S[row j][key 4 g + i], i <
// 4, which is the operand layout that the product O^T += V^T P^T takes its weights
// in, so they never change lanes.  Every wavefront streams keys of its own
// (tiles of 32 keys in 16 bits, 16 in 32): K from memory straight into the MFMA
// operand, a lane 16 bytes of its key's row; V in whole rows into registers,
// which are refilled as soon as their tile is used, so that 16 KiB of a
// wavefront (dim 128) are always under way, without a barrier.  In 16 bits V
// goes through a tile of LDS of the wavefront's own to be read transposed
// (ds_read_b64_tr_b16: in a 16-lane group, lane i receives element i % 4 of the
// 8-byte pieces that lanes 4 e + i / 4 read); in 32 bits a lane's 16 bytes are
// one element each of four MFMA operands, whose columns are dealt accordingly.
// At dim 768 the four wavefronts share their keys and own 192 columns each; the
// shares of the scores are summed through LDS, one barrier a tile.
//
// Keys beyond the last row's reach are read from the last key within it, so that
// nothing is read that no row sees; keys that some rows of a tile do not see get
// the weight zero there.
#pragma once

#include <algorithm>
#include <cmath>

#include "xattn_cache.h"
#include "xattn_launch.h"

namespace xattn {
namespace cache {

constexpr int kRows = 16;      // rows of a work item of cache_attend_kernel
constexpr int kManyRows = 32;  // rows beyond which cache_tile_kernel takes over
constexpr int kWaves = 4;

struct AttendParams {
    Pages pages;
    Batch batch;
    const int* prefix_pages;
    int prefix_len, heads;
    FastDiv group;
    const void* q;
    void* out;
    long long qs, os;
    float c2;         // |scale| log2(e), not zero: scores to base-2 exponents
    unsigned sign;    // flips the sign of q's elements where the scale is negative
    float lag;        // kLag in scores
    int causal;
    int tiles;        // row tiles of a (kv head, range), at most
    int single;       // every sequence has one row tile: tile b is sequence b
    int splits, chunk;  // ranges of keys; split s holds [s * chunk, ...), the last one the rest
    int slot, slots;  // first part of a row that this launch writes, parts of a row
    float* po;        // [token][head][slots][dim] unnormalised
    float2* ml;       // [token][head][slots] (maximum, sum)
};

typedef unsigned int u4 __attribute__((ext_vector_type(4)));
typedef unsigned int u2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;

template <typename T> struct Vec8;
template <> struct Vec8<_Float16> { typedef h8 type; };
template <> struct Vec8<__bf16> { typedef bf8 type; };
template <> struct Vec8<float> { typedef f4 type; };  // not used

template <typename T>
__device__ inline f4 mfma32(u4 a, u4 b, f4 c) {
    typedef typename Vec8<T>::type V;
    if constexpr (__is_same(T, _Float16))
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V, a),
                                                      __builtin_bit_cast(V, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V, a),
                                                       __builtin_bit_cast(V, b), c, 0, 0, 0);
}
// Eight ones: their product with the weights sums them, over all lanes of a row.
template <typename T>
__device__ inline u4 ones() {
    const unsigned two = __is_same(T, __bf16) ? 0x3f803f80u : 0x3c003c00u;
    return u4{two, two, two, two};
}
__device__ inline f4 mfma4(float a, float b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

template <typename T>
__device__ inline unsigned pack2(float lo, float hi) {
    typedef T T2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f2{lo, hi}, T2));
}

// Infinities and NaN in V.  A weight of zero does not silence them in a matrix
// product (0 * inf is NaN), so in tiles that some rows do not see all of they
// are cleared before it; if there were any, those keys are gone through once
// more at the end, and added to the rows that see them as they are: a
// weight is positive, and no finite sum changes what they make of it.
template <typename T>
__device__ inline bool clear_not_finite(u4& x) {
    bool any = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 4) {
            const bool is = (x[e] & 0x7f800000u) == 0x7f800000u;
            any |= is;
            if (is) x[e] = 0;
        } else {
            constexpr unsigned m = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
            const bool lo = (x[e] & m) == m, hi = (x[e] >> 16 & m) == m;
            any |= lo | hi;
            x[e] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
        }
    }
    return any;
}
// Four elements of V with all but infinities and NaN cleared.
template <typename T>
__device__ inline f4 odd_values(const char* v) {
    const Piece4<T> x = *(const Piece4<T>*)v;
    f4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float f = to_f32(x.e[e]);
        y[e] = __builtin_isfinite(f) ? 0.0f : f;
    }
    return y;
}

// A sequence as an item sees it.
struct Sequence {
    int first, end;  // token rows
    int len;         // keys; 0 where it is bad
    bool bad;        // a length that its row of page_table cannot hold
    // Keys that token row t sees.
    __device__ int seen(int t, bool causal) const {
        if (!causal) return len;
        const long long n = (long long)len - (last - t) + 1;
        return n < 0 ? 0 : n < len ? (int)n : len;
    }
    int last;        // q_starts[b + 1], as it is given
};

__device__ inline Sequence sequence(const Batch& B, int b) {
    Sequence s;
    sequence_rows(B, b, &s.first, &s.end);
    s.last = B.q_starts[b + 1];
    s.len = B.kv_lens[b];
    s.bad = s.len < 0 || s.len > B.capacity;
    if (s.bad) s.len = 0;
    return s;
}

// The sequence that row tile `tile` of the batch lies in and its place there,
// last tile first (under a causal mask it has the most keys).  False: none.
template <int ROWS>
__device__ inline bool find_tile(const Batch& B, int group, int tile, int* seq, int* local) {
    const int lane = threadIdx.x % kWave;
    for (int at = 0; at < B.batch; at += kWave) {
        int n = 0;
        if (at + lane < B.batch) {
            int first, end;
            sequence_rows(B, at + lane, &first, &end);
            n = end > first ? (int)(((long long)(end - first) * group + ROWS - 1) / ROWS) : 0;
        }
        int sum = n;
#pragma unroll
        for (int o = 1; o < kWave; o *= 2) {
            const int below = __shfl_up(sum, o);
            if (lane >= o) sum += below;
        }
        const unsigned long long past = __ballot(sum > tile);
        if (past) {
            const int l = __ffsll(past) - 1;
            *seq = at + l;
            *local = __shfl(sum, l) - 1 - tile;
            return true;
        }
        tile -= __shfl(sum, kWave - 1);
    }
    return false;
}

// A work item: rows row0 .. row0 + rows - 1 of a sequence (of the whole batch
// for the prefix) and kv head, and the keys k0 .. k1 - 1.
struct Row {
    int token, head;
};
struct Item {
    Sequence s;
    const int* table;
    unsigned row0, kv_head;
    int rows, split, k0, k1;
    int least;  // keys that all of its rows see
    bool causal;
    __device__ Row row(const AttendParams& p, int i) const {
        const unsigned r = row0 + i, t = p.group.div(r);
        return {s.first + (int)t, (int)(kv_head * p.group.d + r - t * p.group.d)};
    }
    // V's row of a key within k0 .. k1 - 1, of `bytes` bytes; null on a bad page.
    __device__ const char* row_of_v(const AttendParams& p, int k, int bytes) const {
        const unsigned page = p.pages.page_size.div((unsigned)k), size = p.pages.page_size.d;
        const int id = table[page];
        if (id < 0 || (unsigned)id >= p.pages.num_pages) return nullptr;
        return p.pages.v + (size_t)(((unsigned)id * p.pages.kv_heads + kv_head) * size +
                                    ((unsigned)k - page * size)) * bytes;
    }
};

// The workgroup's item; false where it has none.  Row tiles of one kv head and
// key range read the same keys: where those streams deal evenly onto the eight
// XCDs, all tiles of a stream go to one of them and follow each other there, so
// that its L2 reads the keys once.  Otherwise kv heads go fastest and key
// ranges slowest, and of a ragged batch the ranges that few sequences have come
// last.
template <int ROWS, bool PREFIX>
__device__ inline bool find_item(const AttendParams& p, unsigned block, Item* it) {
    unsigned tile, stream;
    const unsigned streams = p.pages.kv_heads * p.splits;
    if (!p.single && streams % kNumXcd == 0) {
        const unsigned at = block / kNumXcd;
        stream = block % kNumXcd + at / p.tiles * kNumXcd;
        tile = at % p.tiles;
        it->kv_head = stream % p.pages.kv_heads;
        it->split = (int)(stream / p.pages.kv_heads);
    } else {
        const unsigned rest = block / p.pages.kv_heads;
        it->kv_head = block % p.pages.kv_heads;
        tile = rest % p.tiles;
        it->split = (int)(rest / p.tiles);
    }
    int local = (int)tile;
    if constexpr (PREFIX) {
        int other;
        sequence_rows(p.batch, 0, &it->s.first, &other);
        sequence_rows(p.batch, p.batch.batch - 1, &other, &it->s.end);
        it->s.len = p.prefix_len;
        it->s.last = 0;
        it->s.bad = false;
        it->table = p.prefix_pages;
    } else {
        int b = (int)tile;
        if (p.single)
            local = 0;
        else if (!find_tile<ROWS>(p.batch, (int)p.group.d, (int)tile, &b, &local))
            return false;
        it->s = sequence(p.batch, b);
        it->table = p.batch.page_table + (long long)b * p.batch.width;
    }
    it->causal = !PREFIX && p.causal;
    // The same in every lane, which the compiler cannot see.
    it->s.first = __builtin_amdgcn_readfirstlane(it->s.first);
    it->s.end = __builtin_amdgcn_readfirstlane(it->s.end);
    it->s.last = __builtin_amdgcn_readfirstlane(it->s.last);
    it->s.len = __builtin_amdgcn_readfirstlane(it->s.len);
    it->s.bad = __builtin_amdgcn_readfirstlane(it->s.bad);
    it->table = uniform_ptr(it->table);
    local = __builtin_amdgcn_readfirstlane(local);
    const long long all = (long long)(it->s.end - it->s.first) * p.group.d;
    const long long row0 = (long long)local * ROWS;
    if (row0 >= all) return false;
    it->row0 = (unsigned)row0;
    it->rows = (int)min((long long)ROWS, all - row0);
    it->least = it->s.seen(it->row(p, 0).token, it->causal);
    const int most = it->s.seen(it->row(p, it->rows - 1).token, it->causal);
    it->k0 = it->split * p.chunk;
    it->k1 = it->split == p.splits - 1 ? most : min(most, it->k0 + p.chunk);
    // Without keys only the first range may have something to store: rows that
    // see nothing, or those of a bad sequence.
    return it->k1 > it->k0 || (it->split == 0 && !PREFIX);
}

// Stores four columns of a row's result: as a part (unnormalised, with its
// maximum and sum) if a merge follows for the row, otherwise as output.
template <typename T, int D, bool PREFIX>
__device__ inline void store(const AttendParams& p, const Item& it, int row, int col, f4 x,
                             float top, float sum) {
    const Row r = it.row(p, row);
    const int n = it.s.seen(r.token, it.causal);
    if (!PREFIX && p.slot == 0 && (p.splits == 1 || n <= p.chunk)) {
        if (it.split > 0) return;
        Piece4<T> y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y.e[e] = (T)(it.s.bad ? NAN : n > 0 ? x[e] / sum : 0.0f);
        *(Piece4<T>*)((T*)p.out + r.token * p.os + (long long)r.head * D + col) = y;
    } else if (it.k0 < n) {
        const size_t at = ((size_t)r.token * p.heads + r.head) * p.slots + p.slot + it.split;
        *(f4*)(p.po + at * D + col) = x;
        if (col == 0) p.ml[at] = {top, sum};
    }
}

template <typename T, int D>
struct Shape {
    static constexpr bool kWide = sizeof(T) == 4;
    static constexpr int kCols = D > 256 ? kWaves : 1;  // wavefronts that share a tile's columns
    static constexpr int kDW = D / kCols;               // columns of a wavefront
    static constexpr int kKeys = kWide ? 16 : 32;       // keys of a tile
    static constexpr int kRegs = kDW / 16;              // 16-byte registers of a lane for K, for V
    static constexpr int kBlocks = kDW / 16;            // 16-column blocks of the output
    static constexpr int kPieces = kDW * (int)sizeof(T) / 16;  // of a row's columns
    static constexpr int kVRow = kDW * 2 + 32;          // bytes of a V row in LDS: 32 of padding
                                                        // deal four rows to distinct banks
    static constexpr int kVTile = kWide ? 0 : kKeys * kVRow;
    static constexpr int kORow = kDW + 4;               // floats of an output row in LDS
    static constexpr int kWaveLds =
        kCols > 1 ? kVTile : (kVTile > kRows * kORow * 4 ? kVTile : kRows * kORow * 4);
    static constexpr int kShare = kKeys * kRows * 4;    // bytes of a wavefront's share of scores
    static constexpr int kStats = kWaves * kRows * 8;   // their maxima and sums
    static constexpr int kLds = kWaves * kWaveLds + (kCols > 1 ? 2 * kWaves * kShare : 0) + kStats;
};

template <typename T, int D, bool PREFIX>
__device__ __forceinline__ void attend_item(const AttendParams& p, unsigned block, char* lds) {
    typedef Shape<T, D> S;
    constexpr int KT = S::kKeys, DW = S::kDW, NR = S::kRegs, NB = S::kBlocks;
    constexpr bool WIDE = S::kWide, SHARED = S::kCols > 1;
    float2(*const stats)[kRows] = (float2(*)[kRows])(lds + S::kLds - S::kStats);
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int j = lane % 16, g = lane / 16;

    Item it;
    if (!find_item<kRows, PREFIX>(p, block, &it)) return;
    const Sequence& s = it.s;
    const int rows = it.rows, least = it.least, k0 = it.k0, k1 = it.k1;
    const unsigned kv_head = it.kv_head;

    // Lane j's row.  Rows behind the last repeat it and are not stored.
    const Row mine = it.row(p, min(j, rows - 1));
    const int seen = min(s.seen(mine.token, it.causal), k1);

    const int col0 = SHARED ? wave * DW : 0;
    u4 qr[NR];
    {
        const T* q = (const T*)p.q + mine.token * p.qs + (long long)mine.head * D + col0;
#pragma unroll
        for (int r = 0; r < NR / (WIDE ? 1 : 2); ++r)
            qr[r] = (WIDE ? *(const u4*)(q + 16 * r + 4 * g) : *(const u4*)(q + 32 * r + 8 * g)) ^
                    p.sign;
    }

    f4 o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = f4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;
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
        return ((ok ? (unsigned)w.id : 0u) * p.pages.kv_heads + kv_head) * p.pages.page_size.d +
               w.slot;
    };
    u4 kr[NR], vr[NR];
    const auto load_k = [&](unsigned row) {
        if constexpr (WIDE) {
            const char* a = p.pages.k + ((size_t)__shfl(row, j) * D + col0) * 4 + 16 * g;
#pragma unroll
            for (int r = 0; r < NR; ++r) kr[r] = *(const u4*)(a + 64 * r);
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const char* a =
                    p.pages.k + ((size_t)__shfl(row, 16 * h + j) * D + col0) * 2 + 16 * g;
#pragma unroll
                for (int r = 0; r < NR / 2; ++r) kr[h * NR / 2 + r] = *(const u4*)(a + 64 * r);
            }
        }
    };
    // V register r of a lane.  32 bits: row 4 g + r % 4, columns 64 (r / 4) + 4 j
    // on.  16 bits: piece 64 r + lane of the tile in row order.
    constexpr int PERIOD = 64 % S::kPieces == 0 ? 1 : S::kPieces / 8;  // registers that end a row
    constexpr int STEP = 64 * PERIOD / S::kPieces;  // ... and the rows they hold
    const auto v_row = [&](int r) {
        return STEP * (r / PERIOD) + ((r % PERIOD) * 64 + lane) / S::kPieces;
    };
    const auto v_piece = [&](int r) { return ((r % PERIOD) * 64 + lane) % S::kPieces; };
    const auto load_v = [&](unsigned row) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            if constexpr (WIDE)
                vr[r] = *(const u4*)(p.pages.v +
                                     ((size_t)__shfl(row, 4 * g + r % 4) * D + col0) * 4 +
                                     256 * (r / 4) + 16 * j);
            else
                vr[r] = *(const u4*)(p.pages.v + ((size_t)__shfl(row, v_row(r)) * D + col0) * 2 +
                                     16 * v_piece(r));
        }
    };

    char* vt = lds + wave * S::kWaveLds;
    const int step = SHARED ? KT : kWaves * KT;
    int k = k0 + (SHARED ? 0 : wave * KT);
    if (k < k1) {
        Where next = find(k);
        const unsigned row = row_of(next);
        next = find(k + step);
        load_k(row);
        load_v(row);
        int turn = 0;
        for (; k < k1; k += step) {
            const bool more = k + step < k1;
            const Where after = find(k + 2 * step);
            // scores
            f4 sc[KT / 16];
#pragma unroll
            for (int h = 0; h < KT / 16; ++h) sc[h] = f4{0, 0, 0, 0};
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                if constexpr (WIDE) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sc[0] = mfma4(__uint_as_float(kr[r][e]), __uint_as_float(qr[r][e]), sc[0]);
                } else {
                    const int h = r % 2, i = r / 2;
                    sc[h] = mfma32<T>(kr[h * NR / 2 + i], qr[i], sc[h]);
                }
            }
            unsigned next_row = 0;
            if (more) {
                next_row = row_of(next);
                load_k(next_row);
            }
            next = after;
            if constexpr (SHARED) {
                char* share = lds + kWaves * S::kWaveLds + (turn & 1) * kWaves * S::kShare;
                turn ^= 1;
#pragma unroll
                for (int h = 0; h < KT / 16; ++h)
                    *(f4*)(share + wave * S::kShare + (h * kWave + lane) * 16) = sc[h];
                lds_barrier();
#pragma unroll
                for (int h = 0; h < KT / 16; ++h) {
                    sc[h] = *(f4*)(share + (h * kWave + lane) * 16);
#pragma unroll
                    for (int w = 1; w < kWaves; ++w)
                        sc[h] += *(f4*)(share + w * S::kShare + (h * kWave + lane) * 16);
                }
            }
            // softmax
            const bool partial = k + KT > least;  // some row does not see all of the tile
            if (partial)
#pragma unroll
                for (int h = 0; h < KT / 16; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (k + 16 * h + 4 * g + i >= seen) sc[h][i] = -INFINITY;
            float top = -INFINITY;
#pragma unroll
            for (int h = 0; h < KT / 16; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[h][i]);
            top = fmaxf(m, wave_max16_groups(top));
            // exponents are taken from 0 while a row has seen nothing
            const float ref = top == -INFINITY ? 0.0f : top * p.c2;
            if (__ballot(top != m)) {
                const float keep = fast_exp2(m * p.c2 - ref);
                l *= keep;
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] *= keep;
                m = top;
            }
#pragma unroll
            for (int h = 0; h < KT / 16; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sc[h][i] = fast_exp2(__builtin_fmaf(sc[h][i], p.c2, -ref));
                    l += sc[h][i];
                }
            // product with V
            if (partial)
#pragma unroll
                for (int r = 0; r < NR; ++r) odd |= clear_not_finite<T>(vr[r]);
            if constexpr (WIDE) {
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[r / 4 * 4 + e] =
                            mfma4(__uint_as_float(vr[r][e]), sc[0][r % 4], o[r / 4 * 4 + e]);
                if (more) load_v(next_row);
            } else {
#pragma unroll
                for (int r = 0; r < NR; ++r)
                    *(u4*)(vt + v_row(r) * S::kVRow + 16 * v_piece(r)) = vr[r];
                if (more) load_v(next_row);
                const u4 w = {pack2<T>(sc[0][0], sc[0][1]), pack2<T>(sc[0][2], sc[0][3]),
                              pack2<T>(sc[1][0], sc[1][1]), pack2<T>(sc[1][2], sc[1][3])};
                lds_s4* at = (lds_s4*)(vt + (4 * g + j / 4) * S::kVRow + j % 4 * 8);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at + 4 * b);
                    const s4 hi =
                        __builtin_amdgcn_ds_read_tr16_b64_v4i16(at + 4 * b + 16 * S::kVRow / 8);
                    const auto both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                    o[b] = mfma32<T>(__builtin_bit_cast(u4, both), w, o[b]);
                }
            }
        }
    }
    if (__ballot(odd))
        for (int t = k0 + (SHARED ? 0 : wave * KT); t < k1; t += step)
            for (int c = t; t + KT > least && c < min(t + KT, k1); ++c)
                if (const char* v = it.row_of_v(p, c, D * (int)sizeof(T)))
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        // 32 bits: element i of block b is column 64 (b / 4) + 16 g + 4 i + b % 4
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

    // Join the wavefronts' parts (of one maximum where they share their keys).
    if (lane < 16) stats[wave][lane] = {m * p.c2, l};
    if constexpr (!SHARED) {
        float* part = (float*)vt + j * S::kORow;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if constexpr (WIDE) {
                // blocks 4 q .. 4 q + 3 hold neighbouring columns
                if (b % 4 == 0)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *(f4*)(part + 16 * b + 16 * g + 4 * i) =
                            f4{o[b][i], o[b + 1][i], o[b + 2][i], o[b + 3][i]};
            } else {
                *(f4*)(part + 16 * b + 4 * g) = o[b];
            }
        }
    }
    __syncthreads();
    if constexpr (SHARED) {
        if (j < rows)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if constexpr (WIDE) {
                    if (b % 4 == 0)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            store<T, D, PREFIX>(p, it, j, col0 + 16 * b + 16 * g + 4 * i,
                                  f4{o[b][i], o[b + 1][i], o[b + 2][i], o[b + 3][i]}, m * p.c2, l);
                } else {
                    store<T, D, PREFIX>(p, it, j, col0 + 16 * b + 4 * g, o[b], m * p.c2, l);
                }
            }
    } else {
        for (int i = threadIdx.x; i < rows * (D / 4); i += 256) {
            const int row = i / (D / 4), col = i % (D / 4) * 4;
            float mx = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, stats[w][row].x);
            const float ref = mx == -INFINITY ? 0.0f : mx;
            f4 x = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float keep = fast_exp2(stats[w][row].x - ref);
                sum += keep * stats[w][row].y;
                x += keep * *(const f4*)((const float*)(lds + w * S::kWaveLds) + row * S::kORow +
                                         col);
            }
            store<T, D, PREFIX>(p, it, row, col, x, mx, sum);
        }
    }
}

// --------------------------------------------------------------------------
// cache_tile_kernel: the same in 16 bits for many rows.  Each of the four
// wavefronts holds RB blocks of sixteen rows, all share tiles of K and V in
// LDS (two of each, filled through registers while the tile before is worked
// on; one barrier a tile).  An operand of K or V read from LDS feeds RB matrix
// instructions.  Weights are taken relative to a maximum that is renewed only
// when a score exceeds it by kLag (in exponents of 2), so that the output is
// rarely rescaled; they stay below 2^kLag, far from the range of either type.
// --------------------------------------------------------------------------
#ifndef WANT_TILE
#define WANT_TILE 4
#define WANT_FEW 2
#define WANT_SINGLE 4
#define WANT_PREFIX 2
#define TILE_STEP 4
#endif
constexpr float kLag = 8.0f;

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
            lds_s4* from = (lds_s4*)(vt + row * LR + 16 * (2 * i + j % 4 / 2 ^ S::swizzle(row)) +
                                     j % 2 * 8);
#pragma unroll
            for (int h = 0; h < KB / 2; ++h) {
                const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(from + 32 * h * LR / 8);
                const s4 hi =
                    __builtin_amdgcn_ds_read_tr16_b64_v4i16(from + (32 * h + 16) * LR / 8);
                const u4 a = __builtin_bit_cast(
                    u4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
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

// --------------------------------------------------------------------------
// Kernels.  The keys of a prefix and those of the sequences are worked on in
// one launch, the prefix's (longer) items first: the sequences' fill in.
// --------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(256) void cache_attend_kernel(AttendParams p) {
    __shared__ __align__(16) char lds[Shape<T, D>::kLds];
    attend_item<T, D, false>(p, blockIdx.x, lds);
}

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void cache_tile_kernel(AttendParams p) {
    __shared__ __align__(16) char lds[TileShape<D>::kLds];
    tile_item<T, D, false>(p, blockIdx.x, lds);
}

// TILES: how many of the two go by tile_item (2: both, 1: the prefix, 0: none).
template <typename T, int D, int TILES>
__global__ __launch_bounds__(256, TILES == 2 || (TILES == 1 && D <= 128) ? 2 : 1) void
cache_prefix_kernel(
    AttendParams prefix, AttendParams own, unsigned prefix_blocks) {
    constexpr int few = TILES < 2 ? Shape<T, D>::kLds : 0;
    constexpr int many = TILES > 0 ? TileShape<D>::kLds : 0;
    __shared__ __align__(16) char lds[few > many ? few : many];
    if (blockIdx.x < prefix_blocks) {
        if constexpr (TILES > 0)
            tile_item<T, D, true>(prefix, blockIdx.x, lds);
        else
            attend_item<T, D, true>(prefix, blockIdx.x, lds);
    } else {
        if constexpr (TILES > 1)
            tile_item<T, D, false>(own, blockIdx.x - prefix_blocks, lds);
        else
            attend_item<T, D, false>(own, blockIdx.x - prefix_blocks, lds);
    }
}

// --------------------------------------------------------------------------
// cache_merge_kernel: out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over the
// parts of a row.  A wavefront takes 256 columns of a row, or all of them, in
// 64 / LANES groups of LANES lanes that take every so many-th part; with
// `together` the four wavefronts of a workgroup share a row's parts (few rows of
// many parts), otherwise each has a row of its own.
// --------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(256) void cache_merge_kernel(AttendParams p, int prefix_parts,
                                                          int together) {
    constexpr int COLS = D > 256 ? 256 : D, LANES = COLS / 4, GROUPS = kWave / LANES;
    __shared__ f4 sums[kWaves - 1][LANES];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const unsigned unit = together ? blockIdx.x : blockIdx.x * kWaves + wave;
    const unsigned row = unit / (D / COLS), col = unit % (D / COLS) * COLS + lane % LANES * 4;
    const int t = (int)(row / p.heads), head = (int)(row % p.heads);
    if (t >= p.batch.tokens) return;
    const int b = token_sequence(p.batch, t);
    if (b >= p.batch.batch) return;
    const Sequence s = sequence(p.batch, b);
    if (t < s.first || t >= s.end) return;
    const int n = s.seen(t, p.causal);
    if (p.slot == 0 && (p.splits == 1 || n <= p.chunk)) return;  // stored already
    const int own = min((n + p.chunk - 1) / p.chunk, p.splits);
    const int parts = prefix_parts + own;
    const size_t at = (size_t)row * p.slots;
    float top = -INFINITY;
    for (int i = lane; i < parts; i += kWave) top = fmaxf(top, p.ml[at + i].x);
    top = wave_max(top);
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    f4 x = {0, 0, 0, 0};
    const int first = lane / LANES + (together ? wave * GROUPS : 0);
    const int step = GROUPS * (together ? kWaves : 1);
    for (int from = 0; from < parts; from += kWave) {
        float weight = 0.0f;
        if (from + lane < parts) {
            const float2 ml = p.ml[at + from + lane];
            weight = fast_exp2(ml.x - ref);
            sum += weight * ml.y;
        }
        const int count = min(kWave, parts - from);
#pragma unroll 4
        for (int i = first; i - first < count; i += step) {
            const int one = min(i, count - 1);
            const float w = __shfl(weight, one);
            const f4 part = *(const f4*)(p.po + (at + from + one) * D + col);
            if (i < count) x += w * part;
        }
    }
    sum = wave_sum(sum);
    if (s.bad) sum = NAN;
#pragma unroll
    for (int o = LANES; o < kWave; o *= 2)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], o);
    if (together) {
        if (wave > 0 && lane < LANES) sums[wave - 1][lane] = x;
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int w = 0; w + 1 < kWaves; ++w) x += sums[w][lane % LANES];
    }
    if (lane < LANES) {
        Piece4<T> y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y.e[e] = (T)(x[e] / sum);
        *(Piece4<T>*)((T*)p.out + t * p.os + (long long)head * D + col) = y;
    }
}

// --------------------------------------------------------------------------
// Plan
// --------------------------------------------------------------------------
struct Range {
    int splits, chunk;
};
constexpr int kMaxSplits = 256;

// Ranges that `keys` keys are divided into where all of them are `items` items of
// work: as many as make `want` workgroups, each of `step` keys or more; with
// several row tiles to a range, of a number that lets the streams deal onto
// the XCDs (find_item).
static Range ranges(long long items, int keys, int step, long long want, int kv, bool single) {
    long long s = std::min<long long>(items > 0 ? want / items : 1, keys / step);
    s = std::max<long long>(1, std::min<long long>(s, kMaxSplits));
    int deal = kNumXcd;
    while (deal > 1 && (long long)kv * deal / 2 % kNumXcd == 0) deal /= 2;
    if (!single && s > deal) s -= s % deal;
    long long chunk = (keys + s - 1) / s;
    chunk = std::max<long long>(step, (chunk + step - 1) / step * step);
    return {single ? (int)std::max<long long>(1, (keys + chunk - 1) / chunk) : (int)s, (int)chunk};
}

struct Plan {
    bool single;            // every sequence has at most sixteen rows
    int rows, prefix_rows;  // rows of a work item
    int tiles, prefix_tiles;
    Range own, prefix;
    int slots() const { return own.splits + prefix.splits; }
    int prefix_parts(int len) const {
        return std::min(prefix.splits, (int)((len + (long long)prefix.chunk - 1) / prefix.chunk));
    }
};

static int tile_rows(int dim) { return dim > 128 ? TileShape<256>::kRows : TileShape<128>::kRows; }

static Plan plan(const Attention& a) {
    Plan p;
    const int kv = (int)a.pages.kv_heads, group = a.heads / kv, dim = a.pages.dim;
    const bool tiled = a.dtype != XATTN_F32 && dim <= 256;  // tile_item takes it
    const int few = (a.dtype == XATTN_F32 ? 16 : 32) * (dim > 256 ? 1 : kWaves);
    const int many = dim > 128 ? TileShape<256>::kKeys : TileShape<128>::kKeys;
    const long long rows = (long long)a.batch.tokens * group, most = (long long)a.max_q * group;
    const long long cu = device_cu_count();
    p.single = most <= kRows;
    p.rows = tiled && most > kManyRows ? tile_rows(dim) : kRows;
    p.tiles = p.single ? a.batch.batch
                       : (int)std::min<long long>(rows / p.rows + a.batch.batch,
                                                  (most + p.rows - 1) / p.rows * a.batch.batch);
    p.own = ranges((long long)p.tiles * kv, a.max_kv, p.rows > kRows ? TILE_STEP * many : few,
                   p.single ? WANT_SINGLE * cu : p.rows > kRows ? WANT_TILE * cu : WANT_FEW * cu, kv, p.single);
    p.prefix_rows = tiled && rows > kManyRows ? tile_rows(dim) : kRows;
    p.prefix_tiles = (int)((rows + p.prefix_rows - 1) / p.prefix_rows);
    p.prefix = a.prefix_len > 0
                   ? ranges((long long)p.prefix_tiles * kv, a.prefix_len,
                            p.prefix_rows > kRows ? TILE_STEP * many : few, WANT_PREFIX * cu, kv, false)
                   : Range{0, 1};
    return p;
}

static size_t parts(const Attention& a, const Plan& p) {
    if (p.prefix.splits == 0 && p.own.splits == 1) return 0;
    return (size_t)a.batch.tokens * a.heads * p.slots();
}

size_t attention_scratch(const Attention& a) {
    return parts(a, plan(a)) * (a.pages.dim * sizeof(float) + sizeof(float2));
}

static unsigned blocks(const AttendParams& p) {
    return p.pages.kv_heads * (unsigned)p.tiles * (unsigned)p.splits;
}

template <typename T, int D>
static void go(const AttendParams& own, const Plan& plan, hipStream_t stream) {
    constexpr bool tiled = sizeof(T) == 2 && D <= 256;
    const bool tile = tiled && plan.rows > kRows, prefix_tile = tiled && plan.prefix_rows > kRows;
    if (plan.prefix.splits > 0) {
        AttendParams p = own;
        p.single = 0;
        p.tiles = plan.prefix_tiles;
        p.splits = plan.prefix.splits;
        p.chunk = plan.prefix.chunk;
        p.slot = 0;
        const unsigned first = blocks(p), all = first + blocks(own);
        if constexpr (tiled) {
            if (tile)
                cache_prefix_kernel<T, D, 2><<<all, 256, 0, stream>>>(p, own, first);
            else if (prefix_tile)
                cache_prefix_kernel<T, D, 1><<<all, 256, 0, stream>>>(p, own, first);
        }
        if (!prefix_tile) cache_prefix_kernel<T, D, 0><<<all, 256, 0, stream>>>(p, own, first);
    } else if (tile) {
        if constexpr (tiled) cache_tile_kernel<T, D><<<blocks(own), 256, 0, stream>>>(own);
    } else {
        cache_attend_kernel<T, D><<<blocks(own), 256, 0, stream>>>(own);
    }
    if (own.po) {
        const long long units = (long long)own.batch.tokens * own.heads * (D > 256 ? D / 256 : 1);
        const bool together = units < 8 * device_cu_count();
        cache_merge_kernel<T, D>
            <<<(unsigned)(together ? units : (units + kWaves - 1) / kWaves), 256, 0, stream>>>(
                own, own.slot, together);
    }
}

template <typename T>
static void by_dim(AttendParams& p, const Plan& plan, hipStream_t stream) {
    if (p.pages.dim == 64) go<T, 64>(p, plan, stream);
    if (p.pages.dim == 128) go<T, 128>(p, plan, stream);
    if (p.pages.dim == 256) go<T, 256>(p, plan, stream);
    if (p.pages.dim == kDim) go<T, kDim>(p, plan, stream);
}

bool launch_attention(const Attention& a, void* scratch, hipStream_t stream) {
    const Plan pl = plan(a);
    AttendParams p{};
    p.pages = a.pages;
    p.batch = a.batch;
    p.prefix_pages = a.prefix_pages;
    p.prefix_len = a.prefix_len;
    p.heads = a.heads;
    p.group = FastDiv::of((unsigned)a.heads / a.pages.kv_heads);
    p.q = a.q;
    p.out = a.out;
    p.qs = a.qs;
    p.os = a.os;
    // A scale of zero makes all scores equal; so does one that is next to it, and a
    // masked score's -infinity stays one.
    p.c2 = std::max(std::fabs(a.scale) * kLog2e, 1e-37f);
    p.lag = std::min(kLag / p.c2, 1e30f);
    p.sign = a.scale >= 0 ? 0 : a.dtype == XATTN_F32 ? 0x80000000u : 0x80008000u;
    p.causal = a.causal;
    p.tiles = pl.tiles;
    p.single = pl.single;
    p.splits = pl.own.splits;
    p.chunk = pl.own.chunk;
    p.slot = pl.prefix_parts(a.prefix_len);
    p.slots = pl.slots();
    if (const size_t n = parts(a, pl)) {
        p.po = (float*)scratch;
        p.ml = (float2*)(p.po + n * a.pages.dim);
    }
    if (a.dtype == XATTN_F32) by_dim<float>(p, pl, stream);
    if (a.dtype == XATTN_F16) by_dim<_Float16>(p, pl, stream);
    if (a.dtype == XATTN_BF16) by_dim<__bf16>(p, pl, stream);
    return check_launch("cache_attend_kernel");
}

}  // namespace cache
}  // namespace xattn
