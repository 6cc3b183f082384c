// What the kernels of cache attention share: their parameters, the work item
// of a workgroup, the matrix instructions' operands, infinities and NaN in V,
// and the store of a result.
#pragma once

#include "xattn_cache.h"

namespace xattn {
namespace cache {

constexpr int kRows = 16;  // rows of a block: a matrix instruction's
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
typedef __attribute__((address_space(3))) u4 lds_u4;
typedef __attribute__((address_space(3))) char lds_char;

template <typename T> struct Vec8;
template <> struct Vec8<_Float16> { typedef h8 type; };
template <> struct Vec8<__bf16> { typedef bf8 type; };

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

// The operand of eight keys of one column, from the 8-byte pieces of four rows at
// `a` and four at `b`.
__device__ inline u4 transposed(const char* a, const char* b) {
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)a);
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)b);
    return __builtin_bit_cast(u4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
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

// The weights of a tile's 32 keys as a matrix operand.
template <typename T>
__device__ inline u4 pack8(f4 lo, f4 hi) {
    return u4{pack2<T>(lo[0], lo[1]), pack2<T>(lo[2], lo[3]), pack2<T>(hi[0], hi[1]),
              pack2<T>(hi[2], hi[3])};
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
// that its L2 reads the keys once (64 rows over 50,176 keys of 768 in 32 bits: 123 us,
// 199 without).  Otherwise kv heads go fastest and key ranges slowest, and of a ragged
// batch the ranges that few sequences have come last.
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
        it->table = p.batch.page_table +
                    (long long)__builtin_amdgcn_readfirstlane(b) * p.batch.width;
    }
    it->causal = !PREFIX && p.causal;
    // The same in every lane, which the compiler cannot see.
    it->s.first = __builtin_amdgcn_readfirstlane(it->s.first);
    it->s.end = __builtin_amdgcn_readfirstlane(it->s.end);
    it->s.last = __builtin_amdgcn_readfirstlane(it->s.last);
    it->s.len = __builtin_amdgcn_readfirstlane(it->s.len);
    it->s.bad = __builtin_amdgcn_readfirstlane(it->s.bad);
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

// One tile of the running softmax of RB rows of lane j: the scores of their keys,
// 4 g + i of each sixteen, become weights relative to a maximum; keys from `seen` on
// (key: that of sc[b][0][0]) weigh nothing.  The maximum m is raised only when a
// score exceeds it by kLag (in exponents of 2), for all rows of the wavefront
// together, so that the output is rarely rescaled: weights stay below 2^kLag, far
// from the range of any type.  l is this lane's share of the sum.  True where
// the output has to be multiplied by `keep`.
constexpr float kLag = 8.0f;

template <int RB, int H>
__device__ inline bool weights(const AttendParams& p, f4 (&sc)[RB][H], bool partial, int key,
                               const int (&seen)[RB], float (&m)[RB], float (&l)[RB],
                               float (&keep)[RB]) {
    if (partial) {
        asm volatile("" : "+v"(key));  // keeps the comparisons in this branch
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int h = 0; h < H; ++h)
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
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) top[b] = fmaxf(top[b], sc[b][h][i]);
        top[b] = wave_max16_groups(top[b]);
        past |= top[b] > m[b] + p.lag;
    }
    const bool raise = __ballot(past) != 0;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        keep[b] = 1.0f;
        if (raise) {
            const float to = fmaxf(m[b], top[b]);
            if (to != m[b]) keep[b] = fast_exp2((m[b] - to) * p.c2);
            m[b] = to;
        }
        // exponents are taken from 0 while a row has seen nothing
        const float ref = m[b] == -INFINITY ? 0.0f : m[b] * p.c2;
        float sum = l[b] * keep[b];
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sc[b][h][i] = fast_exp2(__builtin_fmaf(sc[b][h][i], p.c2, -ref));
                sum += sc[b][h][i];
            }
        l[b] = sum;
    }
    return raise;
}

// Joins the four wavefronts' results of the same rows over keys of their own: their
// maxima and sums in `stats`, their output rows, row_floats apart, in every
// wave_bytes of LDS.
template <typename T, int D, bool PREFIX, int ROWS>
__device__ inline void join_and_store(const AttendParams& p, const Item& it,
                                      const float2 (*stats)[ROWS], const char* lds,
                                      int wave_bytes, int row_floats) {
    for (int i = threadIdx.x; i < it.rows * (D / 4); i += 256) {
        const int row = i / (D / 4), col = i % (D / 4) * 4;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[w][row].x);
        const float ref = top == -INFINITY ? 0.0f : top;
        f4 x = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float keep = fast_exp2(stats[w][row].x - ref);
            sum += keep * stats[w][row].y;
            x += keep * *(const f4*)((const float*)(lds + w * wave_bytes) + row * row_floats + col);
        }
        store<T, D, PREFIX>(p, it, row, col, x, top, sum);
    }
}

}  // namespace cache
}  // namespace xattn
