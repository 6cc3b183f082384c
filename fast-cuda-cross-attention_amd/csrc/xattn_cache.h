// Shared pieces of the cache operators (xattn_rope.h, xattn_cache_attend.h): the
// kernels' views of a paged cache and of a ragged batch, and the look-ups in
// them.  Every look-up is bounded by the host's sizes whatever the device
// arrays hold.
#pragma once

#include "xattn_common.h"

namespace xattn {
namespace cache {

// n / d for 0 <= n < 2^31 by a multiplication: with s = ceil(log2 d) and
// mul = ceil(2^(32 + s) / d) - 2^32, n / d = (mulhi(n, mul) + n) >> s, and the
// sum stays below 2^32.
struct FastDiv {
    unsigned mul, shift, d;
    static FastDiv of(unsigned d) {
        unsigned s = 0;
        while (s < 31 && (1u << s) < d) ++s;
        const unsigned long long p = 1ull << (32 + s);
        return {(unsigned)((p + d - 1) / d - (1ull << 32)), s, d};
    }
    __host__ __device__ unsigned div(unsigned n) const {
        return ((unsigned)(((unsigned long long)n * mul) >> 32) + n) >> shift;
    }
};

// A cache's pages.  A row is one head's dim elements in one slot; rows are
// numbered (page * kv_heads + head) * page_size + slot, below 2^32.
struct Pages {
    char* k;
    char* v;
    unsigned num_pages, kv_heads;
    FastDiv page_size;
    int dim;
};

struct Batch {
    const int* q_starts;
    const int* kv_lens;
    const int* page_table;
    int batch, width, tokens;
    long long capacity;  // positions that a row of page_table can hold
};

struct Rope {
    const double* freqs;
    float amplitude;
    int rot;
    bool interleaved, inverse;
};

constexpr int kMaxRot = 2048;          // rotated elements of a head: their angles fit LDS
constexpr int kMaxKeys = 1 << 30;      // of a sequence or prefix: sums of positions fit an int
constexpr int kMaxBlocks = 0xffffff;   // workgroups of 256 threads in a launch

// Whether a launch of this many workgroups is possible; records the error if not.
inline bool grid_fits(const char* who, long long blocks) {
    if (blocks <= kMaxBlocks) return true;
    set_error(XATTN_ERR_UNSUPPORTED, "%s: a call of %lld workgroups, over %d", who, blocks,
              kMaxBlocks);
    return false;
}

// Launchers; the arguments are valid (xattn_cache_abi.h).
bool launch_rope(const void* x, void* y, const int* positions, const Rope& rope, int dtype,
                 int tokens, int heads, int dim, long long xs, long long ys,
                 hipStream_t stream);
bool launch_append(const Pages& pages, const Batch& batch, const Rope& rope, int dtype,
                   const void* k, long long ks, const void* v, long long vs, const void* q,
                   long long qs, void* q_out, long long qos, int heads, const int* positions,
                   hipStream_t stream);

struct Attention {
    Pages pages;
    Batch batch;
    const int* prefix_pages;
    int prefix_listed, prefix_len;  // 0 keys: no prefix
    int dtype, heads;
    int max_q, max_kv;
    const void* q;
    void* out;
    long long qs, os;
    float scale;
    bool causal;
};
// Bytes of scratch a launch of these sizes takes (the pointers do not count).
size_t attention_scratch(const Attention& a);
bool launch_attention(const Attention& a, void* scratch, hipStream_t stream);

// Four elements of a row.
template <typename T>
struct alignas(4 * sizeof(T)) Piece4 {
    T e[4];
};

// Elements of a cache's type in 32 bits and back (rounded to nearest even).
template <typename T> __device__ inline float to_f32(T x) { return (float)x; }
template <typename T> __device__ inline T from_f32(float x) { return (T)x; }

// Sequence of token row t (wave-uniform; every lane of the wavefront takes
// part): the number of sequences that end at or before t.  May be wrong, but
// not out of 0 .. batch, where q_starts decreases.
__device__ inline int token_sequence(const Batch& B, int t) {
    const int lane = threadIdx.x % kWave;
    int n = 0;
    for (int at = 0; at < B.batch; at += kWave) {
        const int b = at + lane;
        const bool before = b < B.batch && B.q_starts[b + 1] <= t;
        n += __popcll(__ballot(before));
    }
    return n;
}

// Bounds of sequence b's token rows, held within the token tensors.
__device__ inline void sequence_rows(const Batch& B, int b, int* first, int* end) {
    const int lo = B.q_starts[b], hi = B.q_starts[b + 1];
    *first = lo < 0 ? 0 : lo;
    *end = hi > B.tokens ? B.tokens : hi;
}

}  // namespace cache
}  // namespace xattn
