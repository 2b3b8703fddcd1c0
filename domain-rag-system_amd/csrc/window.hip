// Attention with a sliding window and a few first tokens that stay visible, over packed sequences whose keys may be
// kept from earlier calls: self-attention of long documents in local layers, and the few new tokens of a query behind a
// kept prefix.  For encoders with windowed layers, beside the BERT encoders of MedicalEmbedder (reference
// src/indexing/embedder.py:65-71), which have none.  gfx950 only.
//
// Query j of a sequence with nq queries and nk keys stands at position p = nk - nq + j.  It sees key c (0 <= c < nk) if
//   c - p <= right (right < 0: no limit)   and   (p - c <= left (left < 0: no limit)  or  c < n_sinks)
// that is, the keys [0, s) and [lo, hi) of Seen below.  out = sum softmax(scale q.k) v over them; none: 0.
#include "common.h"

#include <algorithm>
#include <atomic>
#include <chrono>
#include <type_traits>

#include <math.h>

namespace {

typedef __bf16 bf16;
typedef _Float16 f16;

template <typename T, int N> struct Vec { typedef T type __attribute__((ext_vector_type(N))); };

struct WinArgs {
    const void *q, *k, *v;
    void* out;
    const int32_t* cu_q;
    const int64_t* k_start;          // NULL: the keys of a sequence are the rows of its queries
    const int32_t* k_len;
    int64_t q_stride, k_row, k_head, v_row, v_head, out_stride;
    int64_t total_q, total_k;
    int32_t n_seq, max_q, max_k, hq, hkv, left, right, sinks;
    float scale;                     // scale * log2(e): the softmax is taken to base 2
};

struct Seq { int64_t q0, k0; int nq, nk; };

// The sequence's rows, checked against the arrays.  False (and flagged): not a sequence of this batch.
__device__ __forceinline__ bool load_seq(const WinArgs& a, int i, Seq& s, uint32_t* fault) {
    s.q0 = a.cu_q[i];
    const int64_t nq = (int64_t)a.cu_q[i + 1] - s.q0;
    int64_t nk = nq;
    s.k0 = s.q0;
    if (a.k_start != nullptr) { s.k0 = a.k_start[i]; nk = a.k_len[i]; }
    const bool q_ok = s.q0 >= 0 && nq >= 0 && nq <= a.max_q && s.q0 <= a.total_q - nq;
    const bool k_ok = s.k0 >= 0 && nk >= 0 && nk <= a.max_k && s.k0 <= a.total_k - nk;
    s.nq = (int)nq;
    s.nk = (int)nk;
    if (!(q_ok && k_ok) && threadIdx.x == 0) rag_flag(fault, q_ok ? RAG_FAULT_KV_ROW : RAG_FAULT_SEGMENT);
    return q_ok && k_ok;
}

struct Seen { int s, lo, hi; };      // visible keys: [0, s) and [lo, hi), s <= lo <= hi

__device__ __forceinline__ Seen seen_by(const WinArgs& a, int p, int nk) {
    Seen w;
    w.hi = a.right < 0 ? nk : max(0, min(nk, p + a.right + 1));
    w.lo = a.left < 0 ? 0 : min(w.hi, max(0, p - a.left));
    w.s = min(a.sinks, w.lo);
    return w;
}

__device__ __forceinline__ bool not_finite(float x) { return !(fabsf(x) < INFINITY); }

// One wave, one query row of one head.  Reads no key and no value that the query does not see, and keeps the mean of the values
// so far instead of their sum, which may be beyond the type's range where the mean is not.
template <typename T, int D>
__device__ void attend_row(const WinArgs& a, const Seq& sq, int j, int head, int lane) {
    typedef typename Vec<T, 8>::type v8;
    constexpr int DL = D / 2;                                // a lane owns 2 dimensions of the result ...
    constexpr int PARTS = 64 / DL;                           // ... of one of these shares of the keys
    const int kvh = head / (a.hq / a.hkv);
    const T* q = reinterpret_cast<const T*>(a.q) + (sq.q0 + j) * a.q_stride + (int64_t)head * D;
    const T* k = reinterpret_cast<const T*>(a.k) + sq.k0 * a.k_row + (int64_t)kvh * a.k_head;
    const T* v = reinterpret_cast<const T*>(a.v) + sq.k0 * a.v_row + (int64_t)kvh * a.v_head;
    const Seen w = seen_by(a, sq.nk - sq.nq + j, sq.nk);
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    const int total = w.s + (w.hi - w.lo);
    const int d0 = 2 * (lane % DL), part = lane / DL;
    for (int base = 0; base < total; base += 64) {
        const int n = min(64, total - base);
        float s = -INFINITY;
        if (lane < n) {
            const int key = base + lane < w.s ? base + lane : base + lane - w.s + w.lo;
            const T* kr = k + (int64_t)key * a.k_row;
            float dot = 0.f;
            for (int d = 0; d < D; d += 8) {
                const v8 kv = *reinterpret_cast<const v8*>(kr + d), qv = *reinterpret_cast<const v8*>(q + d);
#pragma unroll
                for (int e = 0; e < 8; ++e) dot = fmaf((float)kv[e], (float)qv[e], dot);
            }
            s = dot * a.scale;
        }
        float mx = s;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
        const float m_new = fmaxf(m, mx);
        const float top = m_new == -INFINITY ? 0.f : m_new;
        const float p = exp2f(s - top);
        float sum = lane < n ? p : 0.f;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
        const float l_old = l * exp2f(m - top);
        l = l_old + sum;
        m = m_new;
        const float inv = l > 0.f ? 1.f / l : 0.f;
        o0 *= l_old * inv;
        o1 *= l_old * inv;
        for (int i = 0; i < n; i += PARTS) {
            const int mine = i + part;
            const float pi = __shfl(p * inv, min(mine, 63), 64);
            if (mine < n) {
                const int key = base + mine < w.s ? base + mine : base + mine - w.s + w.lo;
                const T* vr = v + (int64_t)key * a.v_row + d0;
                o0 = fmaf(pi, (float)vr[0], o0);
                o1 = fmaf(pi, (float)vr[1], o1);
            }
        }
    }
#pragma unroll
    for (int o = DL; o < 64; o <<= 1) { o0 += __shfl_xor(o0, o, 64); o1 += __shfl_xor(o1, o, 64); }
    if (part == 0) {
        T* dst = reinterpret_cast<T*>(a.out) + (sq.q0 + j) * a.out_stride + (int64_t)head * D + d0;
        dst[0] = (T)(total == 0 ? 0.f : l > 0.f ? o0 : NAN);  // (l: 0 where every score is -infinity, NaN where one is NaN)
        dst[1] = (T)(total == 0 ? 0.f : l > 0.f ? o1 : NAN);
    }
}

// The tiles of `kt` keys that queries j0 .. j1 of a sequence see: `sinks` from the text's start, then `window` from tile w0.
struct Tiles {
    int sinks, w0, n;
    __device__ int first_key(int t, int kt) const { return (t < sinks ? t : w0 + t - sinks) * kt; }
};
__device__ __forceinline__ Tiles tiles_of(const WinArgs& a, const Seq& sq, int j0, int j1, int kt) {
    const Seen first = seen_by(a, sq.nk - sq.nq + j0, sq.nk), last = seen_by(a, sq.nk - sq.nq + j1, sq.nk);
    Tiles t;
    t.sinks = (min(a.sinks, first.lo) + kt - 1) / kt;
    t.w0 = max(t.sinks, first.lo / kt);
    t.n = t.sinks + max(0, (last.hi + kt - 1) / kt - t.w0);
    return t;
}

// How the keys of a call are cut, and where the results of the spans go.
struct FewArgs {
    int chunks;                      // of the workgroups' rows (query * group + head of the group)
    int spans, span;                 // workgroups along the keys, tiles of each
    bool by_seq;                     // a partial result's row: sequence * max_q + query instead of the query's row of q
    float2* part_ml;                 // [row][head][spans]: maximum, sum
    float* part_o;                   // [row][head][spans][D]
    uint64_t* done;                  // [sequence][chunk][key/value head][spans]: `token` where the span's results are written; NULL:
    uint64_t token;                  // window_join_kernel puts them together
};
__device__ __forceinline__ int64_t part_at(const WinArgs& a, const FewArgs& f, const Seq& sq, int seq, int j, int head) {
    return ((f.by_seq ? (int64_t)seq * a.max_q + j : sq.q0 + j) * a.hq + head) * f.spans;
}

// ---- a tile of 128 queries of one head per workgroup ------------------------------------------------------
typedef float f32x16 __attribute__((ext_vector_type(16)));

// 16 neighbouring rows of `pieces` 16-byte pieces, piece p of a row at place p ^ swizzle, cover all banks once at one p
__device__ __forceinline__ int rows_swizzle(int pieces, int row) {
    return pieces >= 16 ? row & 15 : pieces == 8 ? (row >> 1) & 7 : (row >> 2) & 3;
}

// The image of a tile of keys or values in LDS: rows of D 16-bit elements, the 16-byte piece p of row `key` at place
// p ^ swizzle(key), so that neither the rows that a matrix operand reads at one piece nor the blocks that the
// transposing read takes fall on the same banks.  fp32: three such images, of the first, second and third 8 bits of the values.
template <typename E, int D> struct Image {
    static constexpr int PARTS = sizeof(E) == 4 ? 3 : 1;
    static constexpr int ROWB = D * 2;                       // bytes of a row
    static constexpr int PIECES = ROWB / 16;
    static constexpr int KT = sizeof(E) == 4 ? 32 : 64;      // keys of a tile
    static constexpr int PART = KT * ROWB;
    static constexpr int BYTES = PARTS * PART;
    // tiles in LDS at a time: what the registers' occupancy leaves room for
    static constexpr int BUFFERS = sizeof(E) == 4 ? (D == 32 ? 1 : 2) : D == 32 ? 4 : 2;
    static constexpr int WAVES = sizeof(E) == 4 ? (D == 128 ? 1 : D == 64 ? 2 : 4) : (D == 128 ? 2 : D == 64 ? 3 : 4);        // per SIMD
    __device__ static int k_swizzle(int row) { return rows_swizzle(PIECES, row); }
    // 4 neighbouring rows x 4 neighbouring pieces
    __device__ static int v_swizzle(int row) {
        return PIECES == 16 ? (row & 3) << 2 | ((row >> 2) & 3) : PIECES == 8 ? ((row >> 1) & 1) << 2 | ((row >> 2) & 3) : 0;
    }
};

// Two fp32 values as three pairs of bf16, x = x0 + x1 + x2 exactly (8 significant bits each, the rest of every cut is exact)
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& w0, uint32_t& w1, uint32_t& w2) {
    const auto cut = [](float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); };
    const auto high = [](float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u); };
    const float x1 = x - cut(x), y1 = y - cut(y);
    w0 = high(x, y);
    w1 = high(x1, y1);
    w2 = high(x1 - cut(x1), y1 - cut(y1));
}
template <int PARTS, typename V>
__device__ __forceinline__ void split8(const float* v, V* parts) {
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) split_pair(v[2 * i], v[2 * i + 1], w[0][i], w[1][i], w[2][i]);
#pragma unroll
    for (int p = 0; p < PARTS; ++p) parts[p] = V{w[p][0], w[p][1], w[p][2], w[p][3]};
}
// The products of three parts that reach 24 bits, the small ones first
template <typename M, typename F, typename V>
__device__ __forceinline__ F product(const V* x, const V* y, F c) {
    typedef typename M::x8 x8;
    const auto mul = [&](int i, int j) { c = M::mfma(__builtin_bit_cast(x8, x[i]), __builtin_bit_cast(x8, y[j]), c); };
    mul(2, 0); mul(0, 2); mul(1, 1); mul(1, 0); mul(0, 1); mul(0, 0);
    return c;
}

template <typename E> struct Mma;
template <> struct Mma<bf16> {
    typedef typename Vec<bf16, 8>::type x8;
    __device__ static f32x16 mfma(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<f16> {
    typedef typename Vec<f16, 8>::type x8;
    __device__ static f32x16 mfma(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// the lowest n bits (none for n <= 0, all for n >= 32)
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

constexpr float NEG_BIG = -1e30f;    // the running maximum's start: finite, so that no difference of infinities arises
constexpr float LAG = 8.f;           // the maximum may lag behind by this power of two before the sums are rescaled

// Four waves, each 32 queries (the columns of the matrix products) of a 128-query tile of one head; tiles of keys and values
// come into LDS, the next tiles' loads in flight while this one is worked on: 16 bits by direct loads into a ring of two to four,
// fp32 through registers, where they are cut into parts; one barrier a tile (fp32 at head size 32: one buffer, two).
//   S^T = K Q^T        rows = keys, a lane holds 16 keys (registers, lane half) of its query (lane % 32)
//   O^T += V^T P^T     the lane's probabilities are the B operand as they stand; V^T comes out of the row-major image
//                      through the transposing LDS read
// 16-bit types: probabilities are rounded to the type (half a step of each; the result is as far from the exact one again as
// its own rounding takes it), their sum and all other sums are fp32.  In two parts they would cost a second product with the
// values and as much again to cut: 16384 tokens, window 4096, 485 -> 658 us, passages of up to 512 tokens 34.7 -> 40.3.
// fp32: queries, keys, values and probabilities as sums of three bf16 each, exactly; of the nine products the six that reach
// 2^-20 of the factors are taken (the other three stay below 2^-20 together, an fp32 sum over 32 dimensions may be off by 2^-19), all in fp32.
// The matrix cores do six bf16 products in 3/8 of the time of an fp32 one: 4096 tokens, causal, 16 heads of 128 on 8: 411 us,
// with fp32 products 602; 40 sequences of 1 to 512 tokens, 12 heads of 32, window 128: 35.5 and 58.
// The running maximum is raised only when a score exceeds it by more than LAG (the probabilities stay below 2^LAG, in
// the range of every type), so that the rescaling of the sums is rare.
// SPANS: the rows are those of a key/value head (row = query * group + head of the group), the keys are cut as in FewArgs; 4
// sequences of 64 queries, 32 heads of 128 on 8, 4000 to 16000 keys: 72 us (the few-query kernel 165, without spans 250).
// Masked scores are -infinity; a tile that every query of the wave sees whole needs no mask, one that none sees is left
// out.  Where keys or values hold infinities or NaN, 0 * infinity spoils rows that do not see them, and sums of values of
// 1e36 and more may overflow where their mean does not: every row that does not end finite is computed again by attend_row, which
// reads only what the row sees.
// Bound by the matrix cores and the exponentials together: 16384 tokens, 16 heads of 128 on 8, window 4096: 0.48-0.50 ms,
// 0.97-1.0 PFLOP/s (a library product of 8192^3 reaches 1.2); head size 64, no window: 0.36 ms for 2 x 8192, 0.77; float32:
// 167 to 180 TFLOP/s, 1.0 to 1.1 PFLOP/s of bf16 products (a library product in fp32 reaches 0.15).
template <typename E, int D, bool SPANS>
__global__ __launch_bounds__(256, (Image<E, D>::WAVES)) void window_tile_kernel(WinArgs a, FewArgs f, int q_tiles, uint32_t units, bool by_pair, uint32_t* fault) {
    typedef Image<E, D> I;
    typedef typename std::conditional<sizeof(E) == 4, bf16, E>::type M;          // of the matrix operands
    constexpr int KT = I::KT, KB = KT / 32, DT = D / 32, KC = I::PIECES / 2, NB = I::BUFFERS, PARTS = I::PARTS;
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    // All units of a (sequence, key/value head) pair go to workgroups with the same blockIdx % 8, which round-robin
    // placement puts on one XCD: its L2 then holds their keys and values.  Fewer pairs than fill the XCDs evenly: an eighth of
    // the units, neighbours, goes to each instead.  Short pairs' units are turned by one from pair to pair: workgroups go
    // round an XCD's 32 compute units, and where a pair's units divide that number the tiles that only long sequences have would
    // all meet on the same ones (40 sequences of 1 to 512 tokens, 12 heads of 32, float32: 75 us, turned 63).  The last pair is not
    // turned, so that its longest tiles do not end up alone.
    const uint32_t xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
    uint32_t unit = xcd * ((units + 7) >> 3) + at;
    if (by_pair) {
        const uint32_t per_pair = (uint32_t)(a.hq / a.hkv) * (uint32_t)q_tiles, turn = at / per_pair;
        const uint32_t shift = per_pair <= 32 ? (gridDim.x >> 3) / per_pair - 1 - turn : 0;
        unit = (turn * 8 + xcd) * per_pair + (at - turn * per_pair + shift) % per_pair;
    }
    if (unit >= units) return;
    const int group = a.hq / a.hkv;
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int seq, kvh, head, span = 0, first, rows, step;         // the workgroup's rows `first` .. of `rows`: row / step is the query
    if (SPANS) {
        const uint32_t u1 = unit / (uint32_t)f.chunks, u2 = u1 / (uint32_t)f.spans;
        first = (int)(unit - u1 * (uint32_t)f.chunks) * 128;
        span = (int)(u1 - u2 * (uint32_t)f.spans);
        seq = (int)(u2 / (uint32_t)a.hkv);
        kvh = (int)(u2 - (uint32_t)seq * (uint32_t)a.hkv);
        step = group;
    } else {
        const uint32_t u1 = unit / (uint32_t)group, u2 = u1 / (uint32_t)q_tiles;
        first = (q_tiles - 1 - (int)(u1 - u2 * (uint32_t)q_tiles)) * 128;      // (a causal sequence's last tiles are its longest)
        seq = (int)(u2 / (uint32_t)a.hkv);
        kvh = (int)(u2 - (uint32_t)seq * (uint32_t)a.hkv);
        head = kvh * group + (int)(unit - u1 * (uint32_t)group);
        step = 1;
    }
    Seq sq;
    if (!load_seq(a, seq, sq, fault)) return;
    rows = sq.nq * step;
    if (first >= rows) return;

    const int row0 = first + wave * 32, row = row0 + r;      // of the wave, of the lane
    const bool wave_on = row0 < rows, row_on = row < rows;
    const int last_row = rows - 1;
    const auto query = [&](int i) { return SPANS ? min(i, last_row) / step : min(i, last_row); };
    const int qr = query(row);
    if (SPANS) head = kvh * group + min(row, last_row) % step;
    const int shift = sq.nk - sq.nq;                         // position of query 0
    const Seen mine = seen_by(a, shift + qr, sq.nk);
    const Seen w_first = seen_by(a, shift + query(row0), sq.nk), w_last = seen_by(a, shift + query(row0 + 31), sq.nk);
    // the tiles of keys that some query of the workgroup sees
    const Tiles tiles = tiles_of(a, sq, query(first), query(first + 127), KT);
    const int n_spans = SPANS ? max(1, (tiles.n + f.span - 1) / f.span) : 1;
    const int t0 = SPANS ? span * f.span : 0, t1 = SPANS ? min(tiles.n, t0 + f.span) : tiles.n;
    if (SPANS && t0 >= t1 && span > 0) return;

    const unsigned char* kbase = reinterpret_cast<const unsigned char*>(a.k) + (sq.k0 * a.k_row + (int64_t)kvh * a.k_head) * (int64_t)sizeof(E);
    const unsigned char* vbase = reinterpret_cast<const unsigned char*>(a.v) + (sq.k0 * a.v_row + (int64_t)kvh * a.v_head) * (int64_t)sizeof(E);
    const uint32_t k_rowb = (uint32_t)(a.k_row * (int64_t)sizeof(E)), v_rowb = (uint32_t)(a.v_row * (int64_t)sizeof(E));
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
    auto first_key = [&](int t) { return tiles.first_key(t, KT); };
    auto stage = [&](int t) {
        const int key0 = first_key(t);
        const int last = sq.nk - 1 - key0;                   // rows beyond the last key repeat it (masked)
        const unsigned char *kp = kbase + (int64_t)key0 * k_rowb, *vp = vbase + (int64_t)key0 * v_rowb;
        const uint32_t dst = lds0 + (t % NB) * 2 * I::BYTES;
#pragma unroll
        for (int j = 0; j < I::BYTES / 4096; ++j) {
            const int n = wave + 4 * j, o = n * 1024 + lane * 16;
            const int row = o / I::ROWB, place = (o % I::ROWB) / 16;
            const uint32_t src = (uint32_t)min(row, last);
            lds_dma16(dst + n * 1024, kp, src * k_rowb + (place ^ I::k_swizzle(row)) * 16);
            lds_dma16(dst + I::BYTES + n * 1024, vp, src * v_rowb + (place ^ I::v_swizzle(row)) * 16);
        }
    };
    // fp32: rows into registers, from there as three parts into LDS
    constexpr int LOADS = PARTS == 3 ? 2 * KT * I::PIECES / 256 : 1;
    float raw[LOADS][8];
    auto place_of = [&](int j, bool& value, int& row, int& piece) {
        const int n = tid + 256 * j;
        value = n >= KT * I::PIECES;
        row = n / I::PIECES % KT;
        piece = n % I::PIECES;
    };
    auto fetch = [&](int t) {
        const int key0 = first_key(t);
        const int last = sq.nk - 1 - key0;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            bool value;
            int row, piece;
            place_of(j, value, row, piece);
            const unsigned char* p = (value ? vbase : kbase) + (int64_t)key0 * (value ? v_rowb : k_rowb) + (uint32_t)min(row, last) * (value ? v_rowb : k_rowb) + piece * 32;
            const float4 x = reinterpret_cast<const float4*>(p)[0], y = reinterpret_cast<const float4*>(p)[1];
            raw[j][0] = x.x; raw[j][1] = x.y; raw[j][2] = x.z; raw[j][3] = x.w;
            raw[j][4] = y.x; raw[j][5] = y.y; raw[j][6] = y.z; raw[j][7] = y.w;
        }
    };
    auto put = [&](int t) {
        unsigned char* dst = smem + (t % NB) * 2 * I::BYTES;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            bool value;
            int row, piece;
            place_of(j, value, row, piece);
            u32x4 w[3];
            split8<3>(raw[j], w);
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                *reinterpret_cast<u32x4*>(dst + (value ? I::BYTES : 0) + p * I::PART + row * I::ROWB + (piece ^ (value ? I::v_swizzle(row) : I::k_swizzle(row))) * 16) = w[p];
        }
    };
    if (t0 < t1) {
        if constexpr (PARTS == 1) stage(t0);
        else fetch(t0);
    }

    // Q^T: piece 2c + h of the lane's query
    const bool flip = a.scale < 0.f;                         // a negative scale goes into q: the maximum is taken of products as they are
    const float scale = fabsf(a.scale);
    u32x4 qf[KC][PARTS];
    {
        const unsigned char* qp = reinterpret_cast<const unsigned char*>(a.q) + ((sq.q0 + qr) * a.q_stride + (int64_t)head * D) * (int64_t)sizeof(E);
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            if constexpr (PARTS == 1) {
                qf[c][0] = *reinterpret_cast<const u32x4*>(qp + (2 * c + h) * 16);
                if (flip) qf[c][0] ^= 0x80008000u;
            } else {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    v[i] = reinterpret_cast<const float*>(qp)[(2 * c + h) * 8 + i];
                    if (flip) v[i] = -v[i];
                }
                split8<PARTS>(v, qf[c]);
            }
        }
    }
    // (the queries, the last loads so far, are waited for here: later their wait would cover the tiles behind the first too)
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int p = 0; p < PARTS; ++p) asm volatile("" : "+v"(qf[c][p]));
    if constexpr (PARTS == 1) {
#pragma unroll
        for (int t = 1; t < NB - 1; ++t)
            if (t0 + t < t1) stage(t0 + t);
    } else if (NB == 2 && t0 < t1) {
        put(t0);
        if (t0 + 1 < t1) fetch(t0 + 1);
    }
    float m_run = NEG_BIG, l_run = 0.f;                      // l_run: the lane's own keys
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;

    for (int t = t0; t < t1; ++t) {
        if constexpr (PARTS == 1) {
            // this tile's loads; those of the next NB - 2 stay in flight
            if (NB > 2 && t + NB - 2 < t1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"((NB - 2) * (I::BYTES / 2048)) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();                    // every wave has its part, and is done with the tile before
            asm volatile("" ::: "memory");
            if (t + NB - 1 < t1) stage(t + NB - 1);
        } else {
            if (NB == 1) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();                // every wave is done with the tile before
                asm volatile("" ::: "memory");
                put(t);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();                    // the tile is there
            asm volatile("" ::: "memory");
            if (NB == 2 && t + 1 < t1) put(t + 1);
            if (t + NB < t1) fetch(t + NB);
        }
        const int key0 = first_key(t);
        // whether some query of the wave sees some of the tile, and whether all see all of it
        const bool some = wave_on && key0 < w_last.hi && (key0 + KT > w_first.lo || key0 < a.sinks);
        if (!some) continue;
        const bool whole = key0 + KT <= w_first.hi && (key0 >= w_last.lo || key0 + KT <= a.sinks);
        const unsigned char* ks = smem + (t % NB) * 2 * I::BYTES;
        const unsigned char* vs = ks + I::BYTES;
        f32x16 s[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                u32x4 kf[PARTS];
#pragma unroll
                for (int p = 0; p < PARTS; ++p)
                    kf[p] = *reinterpret_cast<const u32x4*>(ks + p * I::PART + (kb * 32 + r) * I::ROWB + ((2 * c + h) ^ I::k_swizzle(r)) * 16);
                if constexpr (PARTS == 1) s[kb] = Mma<M>::mfma(__builtin_bit_cast(typename Mma<M>::x8, kf[0]), __builtin_bit_cast(typename Mma<M>::x8, qf[c][0]), s[kb]);
                else s[kb] = product<Mma<M>>(kf, qf[c], s[kb]);
            }
        }
        if (!whole) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                // a bit per key of the block: [lo, hi) and [0, s)
                const int k0 = key0 + 32 * kb;
                const uint32_t seen = ((below(mine.hi - k0) & ~below(mine.lo - k0)) | below(mine.s - k0)) >> (4 * h);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint32_t keep = (uint32_t)((int32_t)(seen << (31 - (8 * (i >> 2) + (i & 3)))) >> 31);
                    s[kb][i] = __uint_as_float((__float_as_uint(s[kb][i]) & keep) | (0xff800000u & ~keep));
                }
            }
        }
        float mx = NEG_BIG;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
        mx = both_halves_max(mx);
        if (__any((mx - m_run) * scale > LAG)) {
            const float m_new = fmaxf(m_run, mx);
            const float alpha = __builtin_amdgcn_exp2f((m_run - m_new) * scale);
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
        }
        const float ms = m_run * scale;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[kb][i] = __builtin_amdgcn_exp2f(fmaf(s[kb][i], scale, -ms));
                l_run += s[kb][i];
            }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            typedef short tr4 __attribute__((__vector_size__(4 * sizeof(short))));
            const int rho = (lane & 15) >> 2, col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                u32x4 pb[PARTS];
                if constexpr (PARTS == 1) {
                    typename Mma<M>::x8 x;
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = (M)s[kb][8 * tt + j];
                    pb[0] = __builtin_bit_cast(u32x4, x);
                } else {
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = s[kb][8 * tt + j];
                    split8<PARTS>(v, pb);
                }
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    union { tr4 t[2]; u32x4 v; } av[PARTS];
                    u32x4 vf[PARTS];
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const int row = 32 * kb + 16 * tt + 8 * u + 4 * h + rho;
                            const unsigned char* at = vs + p * I::PART + row * I::ROWB + ((dt * 4 + (col >> 3)) ^ I::v_swizzle(row)) * 16 + (col & 4) * 2;
                            av[p].t[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) tr4*)at);
                        }
                        vf[p] = av[p].v;
                    }
                    if constexpr (PARTS == 1) o[dt] = Mma<M>::mfma(__builtin_bit_cast(typename Mma<M>::x8, vf[0]), __builtin_bit_cast(typename Mma<M>::x8, pb[0]), o[dt]);
                    else o[dt] = product<Mma<M>>(vf, pb, o[dt]);
                }
            }
        }
    }
    if (!wave_on) return;

    if (SPANS && n_spans > 1) {
        const float l = both_halves_sum(l_run);
        if (!row_on) return;
        const int64_t at = part_at(a, f, sq, seq, qr, head) + span;
        if (h == 0) f.part_ml[at] = make_float2(m_run, l);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int gq = 0; gq < 4; ++gq)
                *reinterpret_cast<float4*>(f.part_o + at * D + dt * 32 + 8 * gq + 4 * h) = make_float4(o[dt][4 * gq], o[dt][4 * gq + 1], o[dt][4 * gq + 2], o[dt][4 * gq + 3]);
        return;
    }
    const bool any_seen = mine.s + (mine.hi - mine.lo) > 0;
    const float inv = 1.f / both_halves_sum(l_run);
    bool bad = false;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            o[dt][i] = any_seen ? o[dt][i] * inv : 0.f;
            bad |= not_finite(o[dt][i]);
        }
    const uint64_t bad64 = __ballot(bad && row_on);
    const uint32_t bad_rows = (uint32_t)bad64 | (uint32_t)(bad64 >> 32);
    const bool store = row_on && !(bad_rows >> r & 1);
    E* dst = reinterpret_cast<E*>(a.out) + (sq.q0 + qr) * a.out_stride + (int64_t)head * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        if constexpr (sizeof(E) == 4) {
            if (store)
#pragma unroll
                for (int gq = 0; gq < 4; ++gq)
                    *reinterpret_cast<float4*>(dst + dt * 32 + 8 * gq + 4 * h) = make_float4(o[dt][4 * gq], o[dt][4 * gq + 1], o[dt][4 * gq + 2], o[dt][4 * gq + 3]);
        } else {
            // the two lanes of a query trade halves of their groups, so that a lane stores 16 neighbouring bytes
            uint2 grp[4];
#pragma unroll
            for (int gq = 0; gq < 4; ++gq) {
                typename Vec<E, 4>::type v;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = (E)o[dt][4 * gq + j];
                grp[gq] = __builtin_bit_cast(uint2, v);
            }
            trade_halves(grp[0].x, grp[1].x); trade_halves(grp[0].y, grp[1].y);
            trade_halves(grp[2].x, grp[3].x); trade_halves(grp[2].y, grp[3].y);
            if (store) {
                *reinterpret_cast<uint4*>(dst + dt * 32 + 8 * h) = make_uint4(grp[0].x, grp[0].y, grp[1].x, grp[1].y);
                *reinterpret_cast<uint4*>(dst + dt * 32 + 8 * h + 16) = make_uint4(grp[2].x, grp[2].y, grp[3].x, grp[3].y);
            }
        }
    }
    for (uint32_t rest = bad_rows; rest != 0; rest &= rest - 1) {
        const int i = row0 + __builtin_ctz(rest);
        if (SPANS) attend_row<E, D>(a, sq, i / step, kvh * group + i % step, lane);
        else attend_row<E, D>(a, sq, i, head, lane);
    }
}

// ---- few queries over many keys ------------------------------------------------------------------
typedef float f32x4 __attribute__((ext_vector_type(4)));

// The rows of one key/value head's queries (row = query * group + head of the group) are the columns of the matrix
// products, 16 * QT of them per workgroup, so that a key is read once for all of them.  Its waves take tiles of keys in
// turn, each into its own two LDS buffers (no barrier until the end), and put their results together; a long text is cut
// into spans of `span` tiles, one workgroup each, whose results the last of them puts together, or window_join_kernel.
// Probabilities of a 16-bit type: up to 16 rows they are taken in two parts, at 16 bits or more, which costs 0 to 2 % there (one token over
// a window of 1024 8.4 and 8.5 us, 16 tokens on 4000 to 32768 keys 188.8 both); beyond, rounded to the type as above (7 % for 64
// rows).  float32 takes fp32 products, in which nothing is rounded; 64 rows of it at head size 128 are more than the registers
// hold (44 go to scratch).
// Bound by the bytes of the keys and values, 64 KB of them in flight per compute unit at head size 128: 16 tokens over 4000 to
// 32768 kept rows of 8 heads in 0.19 ms, 5.1 TB/s (a large copy moves 4.7).  One token over a window of 1024: 8.4 us, of which the
// launch, the loads of the arguments and the queries, and joining the spans are three quarters.
template <typename E, int D> struct FewImage {
    static constexpr int ROWB = D * (int)sizeof(E);
    static constexpr int PIECES = ROWB / 16;
    static constexpr int KT = sizeof(E) == 4 ? 16 : 32;      // keys of a wave's tile
    static constexpr int BYTES = KT * ROWB;
    static constexpr int NW = 4;                             // waves
    static constexpr size_t lds(int rows) { return (size_t)NW * (4 * BYTES + rows * 8); }
    // waves a SIMD that the LDS leaves room for (kept by the registers too: 23 us for 26 at head size 32 in float32, 64 x 4 queries,
    // window 500), not where 64 rows would spill
    static constexpr int waves(int rows) { return rows <= 32 ? (int)((160 << 10) / (lds(rows) + 1024)) : 1; }
    __device__ static int k_swizzle(int row) { return rows_swizzle(PIECES, row); }
    // 16 bits: 8 neighbouring rows x 2 neighbouring pieces; 32 bits: rows 4 apart, 4 pieces
    __device__ static int v_swizzle(int row) {
        if (sizeof(E) == 4) return PIECES >= 16 ? ((row >> 2) & 3) << 2 : ((row >> 2) & 1) << 2;
        return PIECES == 16 ? (row & 7) << 1 : PIECES == 8 ? ((row >> 1) & 3) << 1 : ((row >> 2) & 1) << 1;
    }
};

template <typename E> struct MmaFew;
template <> struct MmaFew<bf16> {
    __device__ static f32x4 mfma(Mma<bf16>::x8 a, Mma<bf16>::x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct MmaFew<f16> {
    __device__ static f32x4 mfma(Mma<f16>::x8 a, Mma<f16>::x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

__device__ __forceinline__ float quarters_max(float v) {     // over the four lanes that share lane % 16
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
    const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float quarters_sum(float v) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// Values that workgroups on other XCDs read or wrote in the same launch: past the L2, which is an XCD's own.  Results and marks are
// relaxed atomics of agent scope, which this chip writes through and reads past the L2s; their order is that of the hardware
// (a store is counted done by s_waitcnt vmcnt when it has reached memory), not of the language, under which results and
// marks would need a release and an acquire.  Those write back and drop a whole L2 (one token on 4096 keys 19 us for 9.1).
__device__ __forceinline__ void store_through(void* p, float x, float y) {
    const uint64_t v = (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <bool THROUGH>
__device__ __forceinline__ float2 load_pair(const void* p) {
    if (!THROUGH) return *reinterpret_cast<const float2*>(p);
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// One wave: the results of n spans of a query row and head, in the order of the spans.
template <typename E, int D, bool THROUGH>
__device__ void join_row(const WinArgs& a, const FewArgs& f, const Seq& sq, int seq, int j, int head, int n, int lane) {
    const int64_t at = part_at(a, f, sq, seq, j, head);
    const float scale = fabsf(a.scale);
    float top = NEG_BIG;
    for (int i = lane; i < n; i += 64) top = fmaxf(top, load_pair<THROUGH>(f.part_ml + at + i).x);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    constexpr int DL = D / 4, PARTS = 64 / DL;               // four dimensions a lane, PARTS spans at a time
    const int d = (lane % DL) * 4;
    float total = 0.f;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int i = lane / DL; i < n; i += 4 * PARTS) {         // (four spans' loads at once: one by one is a memory latency each)
        float2 p[4], o0[4], o1[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t from = at + min(i + u * PARTS, n - 1);
            p[u] = load_pair<THROUGH>(f.part_ml + from);
            o0[u] = load_pair<THROUGH>(f.part_o + from * D + d);
            o1[u] = load_pair<THROUGH>(f.part_o + from * D + d + 2);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float weight = i + u * PARTS < n ? __builtin_amdgcn_exp2f((p[u].x - top) * scale) : 0.f;
            total += p[u].y * weight;
            sum += f32x4{o0[u].x, o0[u].y, o1[u].x, o1[u].y} * weight;
        }
    }
#pragma unroll
    for (int o = DL; o < 64; o <<= 1) {
        total += __shfl_xor(total, o, 64);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], o, 64);
    }
    const Seen w = seen_by(a, sq.nk - sq.nq + j, sq.nk);
    const bool any_seen = w.s + (w.hi - w.lo) > 0;
    const float inv = 1.f / total;
    typename Vec<E, 4>::type v;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float x = any_seen ? sum[e] * inv : 0.f;
        bad |= not_finite(x);
        v[e] = (E)x;
    }
    if (__any(bad)) attend_row<E, D>(a, sq, j, head, lane);
    else if (lane < DL) *reinterpret_cast<typename Vec<E, 4>::type*>(reinterpret_cast<E*>(a.out) + (sq.q0 + j) * a.out_stride + (int64_t)head * D + d) = v;
}

template <typename E, int D, int QT>
__global__ __launch_bounds__(64 * (FewImage<E, D>::NW), (FewImage<E, D>::waves(16 * QT))) void window_few_kernel(WinArgs a, FewArgs f, uint32_t* fault) {
    typedef FewImage<E, D> I;
    constexpr int KT = I::KT, KB = KT / 16, DT = D / 16, KC = I::PIECES / 4, ROWS = 16 * QT, NW = I::NW;
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];       // [waves][2 buffers][K | V], later [waves][ROWS][D] sums; [waves][ROWS] (m, l)
    const int group = a.hq / a.hkv;
    const uint32_t u1 = blockIdx.x / (uint32_t)a.hkv, u2 = u1 / (uint32_t)f.chunks;
    const int kvh = (int)(blockIdx.x - u1 * (uint32_t)a.hkv), chunk = (int)(u1 - u2 * (uint32_t)f.chunks);
    const int seq = (int)(u2 / (uint32_t)f.spans), span = (int)(u2 - (uint32_t)seq * (uint32_t)f.spans);
    Seq sq;
    if (!load_seq(a, seq, sq, fault)) return;
    const int rows = min(ROWS, sq.nq * group - chunk * ROWS);
    if (rows <= 0) return;
    const int j0 = chunk * ROWS / group, j1 = (chunk * ROWS + rows - 1) / group;
    const Tiles tiles = tiles_of(a, sq, j0, j1, KT);
    const int t0 = span * f.span, t1 = min(tiles.n, t0 + f.span);
    if (t0 >= t1 && span > 0) return;
    const int spans = max(1, (tiles.n + f.span - 1) / f.span);          // that have keys

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const unsigned char* kbase = reinterpret_cast<const unsigned char*>(a.k) + (sq.k0 * a.k_row + (int64_t)kvh * a.k_head) * (int64_t)sizeof(E);
    const unsigned char* vbase = reinterpret_cast<const unsigned char*>(a.v) + (sq.k0 * a.v_row + (int64_t)kvh * a.v_head) * (int64_t)sizeof(E);
    const uint32_t k_rowb = (uint32_t)(a.k_row * (int64_t)sizeof(E)), v_rowb = (uint32_t)(a.v_row * (int64_t)sizeof(E));
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem + wave * 4 * I::BYTES;
    const unsigned char* mine = smem + wave * 4 * I::BYTES;
    constexpr int DMAS = I::BYTES / 1024;
    auto stage = [&](int t, int buf) {
        const int key0 = tiles.first_key(t, KT);
        const int last = sq.nk - 1 - key0;
        const unsigned char *kp = kbase + (int64_t)key0 * k_rowb, *vp = vbase + (int64_t)key0 * v_rowb;
        const uint32_t dst = lds0 + buf * 2 * I::BYTES;
#pragma unroll
        for (int n = 0; n < DMAS; ++n) {
            const int o = n * 1024 + lane * 16;
            const int row = o / I::ROWB, place = (o % I::ROWB) / 16;
            lds_dma16(dst + n * 1024, kp, (uint32_t)min(row, last) * k_rowb + (place ^ I::k_swizzle(row)) * 16);
        }
#pragma unroll
        for (int n = 0; n < DMAS; ++n) {
            const int o = n * 1024 + lane * 16;
            const int row = o / I::ROWB, place = (o % I::ROWB) / 16;
            lds_dma16(dst + I::BYTES + n * 1024, vp, (uint32_t)min(row, last) * v_rowb + (place ^ I::v_swizzle(row)) * 16);
        }
    };

    if (t0 + wave < t1) stage(t0 + wave, 0);
    const bool flip = a.scale < 0.f;
    const float scale = fabsf(a.scale);
    u32x4 qf[QT][KC];
    Seen seen[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int row = chunk * ROWS + min(16 * qt + r, rows - 1), j = row / group, head = kvh * group + row % group;
        seen[qt] = seen_by(a, sq.nk - sq.nq + j, sq.nk);
        const unsigned char* qp = reinterpret_cast<const unsigned char*>(a.q) + ((sq.q0 + j) * a.q_stride + (int64_t)head * D) * (int64_t)sizeof(E);
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            qf[qt][c] = *reinterpret_cast<const u32x4*>(qp + (4 * c + g) * 16);
            if (flip) qf[qt][c] ^= sizeof(E) == 4 ? 0x80000000u : 0x80008000u;
        }
    }
    float m[QT], l[QT];
    f32x4 o[QT][DT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        m[qt] = NEG_BIG;
        l[qt] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[qt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // (the queries, the last loads so far, are waited for here: inside the loop their wait would cover the next tile too)
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int c = 0; c < KC; ++c) asm volatile("" : "+v"(qf[qt][c]));
    for (int t = t0 + wave, buf = 0; t < t1; t += NW, buf ^= 1) {
        if (t + NW < t1) {
            stage(t + NW, buf ^ 1);
            asm volatile("s_waitcnt vmcnt(%0)" :: "n"(2 * DMAS) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        const int key0 = tiles.first_key(t, KT);
        const unsigned char* ks = mine + buf * 2 * I::BYTES;
        const unsigned char* vs = ks + I::BYTES;
        f32x4 s[QT][KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) s[qt][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const u32x4 kf = *reinterpret_cast<const u32x4*>(ks + (kb * 16 + r) * I::ROWB + ((4 * c + g) ^ I::k_swizzle(kb * 16 + r)) * 16);
#pragma unroll
                for (int qt = 0; qt < QT; ++qt) {
                    if constexpr (sizeof(E) == 4) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            s[qt][kb] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf[j]), __uint_as_float(qf[qt][c][j]), s[qt][kb], 0, 0, 0);
                    } else {
                        s[qt][kb] = MmaFew<E>::mfma(__builtin_bit_cast(typename Mma<E>::x8, kf), __builtin_bit_cast(typename Mma<E>::x8, qf[qt][c]), s[qt][kb]);
                    }
                }
            }
        }
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            float mx = NEG_BIG;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + 16 * kb + 4 * g + i;
                    const bool ok = key < seen[qt].hi && (key >= seen[qt].lo || key < seen[qt].s);
                    s[qt][kb][i] = ok ? s[qt][kb][i] : -INFINITY;
                    mx = fmaxf(mx, s[qt][kb][i]);
                }
            mx = quarters_max(mx);
            if (__any((mx - m[qt]) * scale > LAG)) {
                const float m_new = fmaxf(m[qt], mx);
                const float alpha = __builtin_amdgcn_exp2f((m[qt] - m_new) * scale);
                m[qt] = m_new;
                l[qt] *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[qt][dt][i] *= alpha;
            }
            const float ms = m[qt] * scale;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[qt][kb][i] = __builtin_amdgcn_exp2f(fmaf(s[qt][kb][i], scale, -ms));
                    l[qt] += s[qt][kb][i];
                }
        }
        if constexpr (sizeof(E) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = 4 * g + i;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const float v = *reinterpret_cast<const float*>(vs + key * I::ROWB + (((dt * 4 + (r >> 2)) ^ I::v_swizzle(key)) * 16) + (r & 3) * 4);
#pragma unroll
                    for (int qt = 0; qt < QT; ++qt) o[qt][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, s[qt][0][i], o[qt][dt], 0, 0, 0);
                }
            }
        } else {
            typedef short tr4 __attribute__((__vector_size__(4 * sizeof(short))));
            constexpr bool TWO = QT == 1;                     // probabilities as the type's value and what it leaves
            typename Mma<E>::x8 pb[QT], rest[QT];
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float p = s[qt][(j >> 2) % KB][j & 3];
                    pb[qt][j] = (E)p;
                    if (TWO) rest[qt][j] = (E)(p - (float)pb[qt][j]);
                }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                union { tr4 t[2]; typename Mma<E>::x8 v; } av;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int row = 16 * u + 4 * g + (r >> 2);
                    const unsigned char* p = vs + row * I::ROWB + (((dt * 2 + ((r & 3) >> 1)) ^ I::v_swizzle(row)) * 16) + (r & 1) * 8;
                    av.t[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) tr4*)p);
                }
#pragma unroll
                for (int qt = 0; qt < QT; ++qt) {
                    if (TWO) o[qt][dt] = MmaFew<E>::mfma(av.v, rest[qt], o[qt][dt]);
                    o[qt][dt] = MmaFew<E>::mfma(av.v, pb[qt], o[qt][dt]);
                }
            }
        }
    }

    // the waves' results side by side in LDS (each over its own buffers), then one value per thread and step
    float* sums = reinterpret_cast<float*>(smem);
    constexpr int WAVE_F = I::BYTES;                          // floats of a wave's buffers: 4 * BYTES / 4
    static_assert(WAVE_F >= ROWS * D, "a wave's sums fit its buffers");
    float2* ml = reinterpret_cast<float2*>(smem + NW * 4 * I::BYTES);
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const float ls = quarters_sum(l[qt]);
        if (g == 0) ml[wave * ROWS + 16 * qt + r] = make_float2(m[qt], ls);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(sums + wave * WAVE_F + (16 * qt + r) * D + dt * 16 + 4 * g) = o[qt][dt];
    }
    __syncthreads();
    __shared__ uint32_t bad_rows[2];
    if (tid < 2) bad_rows[tid] = 0;
    __syncthreads();
    for (int i = tid; i < rows * (D / 4); i += 64 * NW) {
        const int lr = i / (D / 4), d = (i % (D / 4)) * 4;
        const int row = chunk * ROWS + lr, j = row / group, head = kvh * group + row % group;
        float top = NEG_BIG;
#pragma unroll
        for (int w = 0; w < NW; ++w) top = fmaxf(top, ml[w * ROWS + lr].x);
        float total = 0.f;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float2 p = ml[w * ROWS + lr];
            const float weight = __builtin_amdgcn_exp2f((p.x - top) * scale);
            total += p.y * weight;
            sum += *reinterpret_cast<const f32x4*>(sums + w * WAVE_F + lr * D + d) * weight;
        }
        if (spans > 1) {
            const int64_t at = part_at(a, f, sq, seq, j, head) + span;
            if (d == 0) store_through(f.part_ml + at, top, total);
            store_through(f.part_o + at * D + d, sum[0], sum[1]);
            store_through(f.part_o + at * D + d + 2, sum[2], sum[3]);
        } else {
            const Seen w = seen_by(a, sq.nk - sq.nq + j, sq.nk);
            const bool any_seen = w.s + (w.hi - w.lo) > 0;
            const float inv = 1.f / total;
            typename Vec<E, 4>::type v;
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = any_seen ? sum[e] * inv : 0.f;
                bad |= not_finite(x);
                v[e] = (E)x;
            }
            if (bad) atomicOr(&bad_rows[lr >> 5], 1u << (lr & 31));
            *reinterpret_cast<typename Vec<E, 4>::type*>(reinterpret_cast<E*>(a.out) + (sq.q0 + j) * a.out_stride + (int64_t)head * D + d) = v;
        }
    }
    if (spans > 1) {
        // The workgroup that finds the results of all spans written puts them together.  If two find it, both store the same values.  The
        // marks may hold anything before the call: its token is none that an earlier call left, and they are cleared after use,
        // so that a captured call finds them cleared when it runs again.
        if (f.done == nullptr) return;
        __shared__ int all;
        uint64_t* done = f.done + ((int64_t)(seq * f.chunks + chunk) * a.hkv + kvh) * f.spans;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                // every thread's results are written, before ...
        __syncthreads();
        if (wave == 0) {
            if (lane == 0) __hip_atomic_store(done + span, f.token, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");            // ... the mark, before the marks are read: the last one finds all
            bool here = true;
            for (int i = lane; i < spans; i += 64) here &= __hip_atomic_load(done + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == f.token;
            const bool yes = __all(here);
            if (yes)
                for (int i = lane; i < spans; i += 64) __hip_atomic_store(done + i, (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (lane == 0) all = yes;
        }
        __syncthreads();
        if (!all) return;
        for (int lr = wave; lr < rows; lr += NW) {
            const int row = chunk * ROWS + lr;
            join_row<E, D, true>(a, f, sq, seq, row / group, kvh * group + row % group, spans, lane);
        }
        return;
    }
    __syncthreads();                                         // (also: the rows' stores are done before a row is written again)
    for (int lr = wave; lr < rows; lr += NW)
        if (bad_rows[lr >> 5] >> (lr & 31) & 1) {
            const int row = chunk * ROWS + lr;
            attend_row<E, D>(a, sq, row / group, kvh * group + row % group, lane);
        }
}

// The results of one query row and head whose chunks of rows are not put together by window_few_kernel, a wave each.
template <typename E, int D>
__global__ __launch_bounds__(256) void window_join_kernel(WinArgs a, FewArgs f, int rows_of_chunk, int kt) {
    const int group = a.hq / a.hkv, lane = threadIdx.x & 63;
    const int per_seq = (a.max_q * a.hq + 3) / 4;
    const int seq = (int)(blockIdx.x / per_seq);
    const int id = (int)(blockIdx.x % per_seq) * 4 + (int)(threadIdx.x >> 6);
    const int j = id / a.hq, head = id % a.hq;
    Seq sq;
    if (!load_seq(a, seq, sq, nullptr) || j >= sq.nq) return;
    const int chunk = (j * group + head % group) / rows_of_chunk;
    const int last = min((chunk + 1) * rows_of_chunk, sq.nq * group) - 1;
    const Tiles tiles = tiles_of(a, sq, chunk * rows_of_chunk / group, last / group, kt);
    const int n = (tiles.n + f.span - 1) / f.span;
    if (n > 1) join_row<E, D, false>(a, f, sq, seq, j, head, n, lane);          // (one span's results are stored as they are)
}

// How a call runs, from its sizes alone (the workspace is computed from the same).
enum Kernel { TILE, FEW, TILE_SPANS };
struct Plan {
    Kernel kernel;
    int qt, chunks, spans, span;     // 16-row columns of a workgroup (few), chunks of the rows, spans along the keys
    int64_t parts;                   // query rows * heads * spans whose partial results the workspace holds
    int64_t marks;                   // 0: window_join_kernel puts them together
    int64_t bytes(int D) const { return marks * 8 + parts * (D + 2) * 4; }
};

// The most keys that `queries` neighbouring queries can see, in tiles of kt
int64_t most_tiles(int max_k, int queries, int left, int right, int sinks, int kt) {
    int64_t keys = max_k;
    if (left >= 0) keys = std::min<int64_t>(keys, (int64_t)sinks + left + queries + (right < 0 ? max_k : std::min(right, max_k)));
    return std::max<int64_t>(1, (keys + kt - 1) / kt + (left >= 0 ? 2 : 0));
}

Plan plan_of(int64_t total_q, int n_seq, int max_q, int max_k, int hq, int hkv, int D, int left, int right, int sinks, int size) {
    const int group = hq / hkv, wide = size == 4, di = D == 32 ? 0 : D == 64 ? 1 : 2;
    const int64_t rows = (int64_t)max_q * group, pairs = std::min<int64_t>(1 << 24, (int64_t)n_seq * hkv);      // (caps: no overflow below)

    // Which kernel: the times estimated in microseconds.  The tile kernel walks the keys of 128 queries one tile after the
    // other; with spans it takes the rows of a key/value head together and spreads them and their keys over the chip, with a second
    // launch; the few-query kernel spreads them too but reads them once per 64 rows, with narrower matrix operands.  The
    // constants are fitted to the kernels' times over 197 sizes a type and head size (1 to 32 sequences, 9 to 1500 queries, 600 to
    // 16384 keys); the chosen times are 1 % over the best of the three on average, without the spans 30 %.  E.g. head size 128,
    // bf16, 16 heads on 8, 4 sequences of 200 queries on 4096 keys: few 102 us, spans 58, tiles 91; of 9 queries: 24, 23, 85.
    static const double few_tile[2][3] = {{1.0, 1.0, 1.7}, {1.0, 2.4, 3.4}};            // of 17 to 32 rows
    static const double one_tile[2][3] = {{0.9, 0.9, 1.0}, {0.9, 1.5, 1.8}}, all_tiles[2][3] = {{0.7, 0.7, 1.07}, {0.7, 1.3, 1.8}};
    static const int on_cu[2][3] = {{4, 3, 2}, {4, 2, 1}};   // workgroups of the tile kernel
    const auto tile_time = [&](int64_t tiles, double wgs, int64_t rows_of_wg) {
        return (double)tiles * std::max(one_tile[wide][di], all_tiles[wide][di] * wgs * std::min<int64_t>(4, (rows_of_wg + 31) / 32 + 1) / 1024);
    };
    Plan tile{}, few{}, cut{};
    const int kt_tile = wide ? 32 : 64;
    const double tile_us = 9 + tile_time(most_tiles(max_k, std::min(max_q, 128), left, right, sinks, kt_tile), (double)n_seq * hq * ((max_q + 127) / 128), max_q);

    few.kernel = FEW;
    few.qt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    few.chunks = (int)std::min<int64_t>(1 << 24, (rows + 16 * few.qt - 1) / (16 * few.qt));
    const int kt = wide ? 16 : 32;
    const int64_t tiles = most_tiles(max_k, max_q, left, right, sinks, kt), base = std::min<int64_t>(1 << 24, pairs * few.chunks);
    const double few_us = (few.qt == 4 ? 18 : 9) + (double)base * tiles / 1024 * few_tile[wide][di] * (few.qt == 4 ? 2.1 : few.qt == 1 && wide ? 0.5 : 1);

    cut.kernel = TILE_SPANS;
    cut.chunks = (int)std::min<int64_t>(1 << 24, (rows + 127) / 128);
    const int64_t cut_tiles = most_tiles(max_k, (int)std::min<int64_t>(max_q, 127 / group + 2), left, right, sinks, kt_tile);
    const int64_t cut_base = std::min<int64_t>(1 << 24, pairs * cut.chunks), cut_cuts = std::max<int64_t>(1, 256 * on_cu[wide][di] / cut_base);
    cut.span = (int)std::max<int64_t>(8, (cut_tiles + cut_cuts - 1) / cut_cuts);
    cut.spans = (int)((cut_tiles + cut.span - 1) / cut.span);
    cut.parts = cut.spans > 1 ? std::min(total_q, (int64_t)n_seq * max_q) * hq * cut.spans : 0;
    double cut_us = (cut.spans > 1 ? 15 : 9) + tile_time(std::min<int64_t>(cut.span, cut_tiles), (double)cut_base * cut.spans, rows) +
                    (double)cut.parts * (D + 2) / 1e6;       // (8 bytes each, written and read)
    if (rows <= 16) cut_us = tile_us;                        // columns of the matrix products mostly empty (16 sequences of unlike lengths, one
                                                             // token: 227 us, few 188)
    if (few_us >= std::min(tile_us, cut_us) || base == 1 << 24) return cut_us < 0.9 * tile_us && cut_base < 1 << 24 ? cut : tile;
    Plan& p = few;

    // A workgroup's start, the filling of its buffers and its end cost as much as some 8 tiles a wave, so the workgroups that are on
    // the chip at once (256 compute units by what their LDS leaves room for) run one round: one token over 32768 keys of 8 heads
    // 36.6 us, in two rounds 44, in three 51.  Spans that would be long all the same (over 256 tiles) are cut in three, against
    // sequences of unlike lengths: 16 sequences of 4000 to 32768 keys 223 -> 190 us.  Spans of 4 tiles, a wave's one, are the
    // shortest while they are few, 8 from 128 tiles on (one token, head size 128: 1024 keys in spans of 4 7.6 us, 8 8.6, 12 9.6; 4096
    // keys 9.8, 9.2, 10.6).  One span, where joining costs more than it gives, by what its tiles take (512 keys: one span 8.1
    // us, spans of 4 7.8, at head size 64 6.4 and 6.8; 200 keys in float32: 10.5 and 8.4).
    const int64_t on_chip = 256 * ((160 << 10) / (16 * (int64_t)kt * D * size + 2048));
    int64_t cuts = std::max<int64_t>(1, on_chip / base);
    if (tiles / cuts > 256) cuts = std::max<int64_t>(1, 3 * on_chip / base);
    const int64_t one_span = std::min(20, (wide ? 768 : 2048) / D), shortest = std::min<int64_t>(8, std::max<int64_t>(4, tiles / 16));
    p.span = (int)(tiles <= one_span ? tiles : std::max(shortest, (tiles + cuts - 1) / cuts));
    p.spans = (int)((tiles + p.span - 1) / p.span);
    p.parts = p.spans > 1 ? std::min(total_q, (int64_t)n_seq * max_q) * hq * p.spans : 0;
    // Joined by the workgroups themselves, a row each wave, where that is the shorter (one token of 4 heads on one, head size 128:
    // 1024 keys 8.8 us, with the second launch 9.4; 65536 keys, 256 spans, 28.5 and 26.1; 8 rows on 1024 keys 10.6 and 9.8) or saves
    // a launch of the host's 4 us at no more than 6 % (16384 keys, 64 spans: 13.0 us and 12.3).
    if (p.spans > 1 && rows <= 4 && p.spans <= 64) p.marks = ((int64_t)n_seq * p.chunks * hkv * p.spans + 1) / 2 * 2;
    return p;
}

FewArgs few_args(const WinArgs& a, const Plan& p, int D, void* work) {
    static std::atomic<uint64_t> tokens{(uint64_t)std::chrono::steady_clock::now().time_since_epoch().count() * 0x9e3779b97f4a7c15ull | 1};
    FewArgs f;
    f.chunks = p.chunks; f.spans = p.spans; f.span = p.span;
    f.by_seq = (int64_t)a.n_seq * a.max_q < a.total_q;       // rows of no sequence take no room
    f.done = p.marks > 0 ? reinterpret_cast<uint64_t*>(work) : nullptr;
    f.token = p.marks > 0 ? tokens.fetch_add(2) : 0;         // (odd: never what a call leaves)
    f.part_o = reinterpret_cast<float*>(reinterpret_cast<uint64_t*>(work) + p.marks);
    f.part_ml = reinterpret_cast<float2*>(f.part_o + p.parts * D);
    return f;
}

template <typename T, int D>
int window_join(const WinArgs& a, const FewArgs& f, int rows_of_chunk, int kt, hipStream_t stream) {
    const int64_t joins = (int64_t)a.n_seq * (((int64_t)a.max_q * a.hq + 3) / 4);
    RAG_REQUIRE(joins < (1ll << 24), RAG_ELIMIT, "rag_enc_attention_window: too many query rows");
    window_join_kernel<T, D><<<(unsigned)joins, 256, 0, stream>>>(a, f, rows_of_chunk, kt);
    RAG_HIP_TRY(hipGetLastError());
    return RAG_OK;
}

template <typename T, int D, int QT>
int window_few(const WinArgs& a, const Plan& p, void* work, hipStream_t stream) {
    const FewArgs f = few_args(a, p, D, work);
    const int64_t grid = (int64_t)a.n_seq * p.spans * p.chunks * a.hkv;
    RAG_REQUIRE(grid < (1ll << 24), RAG_ELIMIT, "rag_enc_attention_window: too many sequences");
    constexpr size_t lds = FewImage<T, D>::lds(16 * QT);
    RAG_GRANT_LDS((window_few_kernel<T, D, QT>), lds);
    window_few_kernel<T, D, QT><<<(unsigned)grid, 64 * FewImage<T, D>::NW, lds, stream>>>(a, f, rag_fault_word());
    RAG_HIP_TRY(hipGetLastError());
    return p.spans > 1 && p.marks == 0 ? window_join<T, D>(a, f, 16 * QT, FewImage<T, D>::KT, stream) : RAG_OK;
}

template <typename T, int D>
int window_launch(const WinArgs& a, void* work, int64_t work_bytes, hipStream_t stream) {
    const Plan p = plan_of(a.total_q, a.n_seq, a.max_q, a.max_k, a.hq, a.hkv, D, a.left, a.right, a.sinks, (int)sizeof(T));
    RAG_REQUIRE(p.bytes(D) <= work_bytes, RAG_EINVAL, "rag_enc_attention_window: the workspace holds %lld bytes, %lld are needed",
                (long long)work_bytes, (long long)p.bytes(D));
    if (p.kernel == FEW) {
        if (p.qt == 1) return window_few<T, D, 1>(a, p, work, stream);
        if (p.qt == 2) return window_few<T, D, 2>(a, p, work, stream);
        return window_few<T, D, 4>(a, p, work, stream);
    }
    constexpr size_t lds = 2 * (size_t)Image<T, D>::BUFFERS * Image<T, D>::BYTES;
    const int64_t pairs = (int64_t)a.n_seq * a.hkv;
    if (p.kernel == TILE_SPANS) {
        const FewArgs f = few_args(a, p, D, work);
        const int64_t units = pairs * p.chunks * p.spans, grid = (units + 7) / 8 * 8;
        RAG_REQUIRE(grid < (1ll << 24), RAG_ELIMIT, "rag_enc_attention_window: too many query tiles");
        RAG_GRANT_LDS((window_tile_kernel<T, D, true>), lds);
        window_tile_kernel<T, D, true><<<(unsigned)grid, 256, lds, stream>>>(a, f, 0, (uint32_t)units, false, rag_fault_word());
        RAG_HIP_TRY(hipGetLastError());
        return p.spans > 1 ? window_join<T, D>(a, f, 128, Image<T, D>::KT, stream) : RAG_OK;
    }
    const int q_tiles = (a.max_q + 127) / 128;
    const int64_t units = pairs * q_tiles * (a.hq / a.hkv);
    const bool by_pair = pairs % 8 == 0 || pairs >= 64;
    const int64_t grid = by_pair ? (pairs + 7) / 8 * 8 * q_tiles * (a.hq / a.hkv) : (units + 7) / 8 * 8;
    RAG_REQUIRE(grid < (1ll << 24), RAG_ELIMIT, "rag_enc_attention_window: too many query tiles");
    RAG_GRANT_LDS((window_tile_kernel<T, D, false>), lds);
    window_tile_kernel<T, D, false><<<(unsigned)grid, 256, lds, stream>>>(a, FewArgs{}, q_tiles, (uint32_t)units, by_pair, rag_fault_word());
    RAG_HIP_TRY(hipGetLastError());
    return RAG_OK;
}

template <typename T>
int window_by_dim(const WinArgs& a, int D, void* work, int64_t work_bytes, hipStream_t stream) {
    if (D == 32) return window_launch<T, 32>(a, work, work_bytes, stream);
    if (D == 64) return window_launch<T, 64>(a, work, work_bytes, stream);
    return window_launch<T, 128>(a, work, work_bytes, stream);
}

constexpr int FAR = 1 << 30;         // a window beyond every length is no limit (and positions never overflow)

}  // namespace

extern "C" int64_t rag_enc_attention_window_workspace(int64_t total_q, int32_t n_seq, int32_t max_q_len, int32_t max_k_len,
                                                      int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                                      int32_t window_left, int32_t window_right, int32_t n_sinks, int32_t dtype) {
    if (total_q <= 0 || n_seq <= 0 || max_q_len <= 0 || max_k_len < 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads || head_dim <= 0 ||
        n_sinks < 0 || window_left < -1 || window_right < -1)
        return 0;                                            // nothing to run, or refused by the call
    const Plan p = plan_of(total_q, n_seq, max_q_len, max_k_len, n_q_heads, n_kv_heads, head_dim, window_left >= FAR ? -1 : window_left,
                           window_right >= FAR ? -1 : window_right, n_sinks, dtype == RAG_DTYPE_F32 ? 4 : 2);
    return p.bytes(head_dim);
}

extern "C" int rag_enc_attention_window_dev(const void* d_q, int64_t q_stride, const void* d_k, int64_t k_row_stride,
                                            int64_t k_head_stride, const void* d_v, int64_t v_row_stride, int64_t v_head_stride,
                                            const int32_t* d_cu_q, int64_t total_q, const int64_t* d_k_start,
                                            const int32_t* d_k_len, int64_t total_k, int32_t n_seq, int32_t max_q_len,
                                            int32_t max_k_len, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, float scale,
                                            int32_t window_left, int32_t window_right, int32_t n_sinks, int32_t dtype, void* d_out,
                                            int64_t out_stride, void* d_workspace, int64_t workspace_bytes, void* stream_) {
    const char* me = "rag_enc_attention_window";
    RAG_REQUIRE(dtype == RAG_DTYPE_F32 || dtype == RAG_DTYPE_BF16 || dtype == RAG_DTYPE_F16, RAG_EINVAL, "%s: unknown dtype %d", me, dtype);
    RAG_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128, RAG_ELIMIT, "%s: head_dim must be 32, 64 or 128 (got %d)", me, head_dim);
    RAG_REQUIRE(n_seq >= 0 && max_q_len >= 0 && max_k_len >= 0 && total_q >= 0 && total_k >= 0, RAG_EINVAL, "%s: bad sizes", me);
    RAG_REQUIRE(total_q < (1ll << 31) && max_q_len < (1 << 30) && max_k_len < (1 << 30), RAG_ELIMIT, "%s: sizes beyond the limit", me);
    RAG_REQUIRE(n_kv_heads >= 1 && n_q_heads >= 1 && n_q_heads <= 4096 && n_q_heads % n_kv_heads == 0, RAG_EINVAL,
                "%s: the query heads must be a multiple of the key/value heads", me);
    RAG_REQUIRE(window_left >= -1 && window_right >= -1 && n_sinks >= 0, RAG_EINVAL, "%s: bad window", me);
    RAG_REQUIRE(isfinite(scale * 1.4426950408889634f), RAG_EINVAL, "%s: bad scale", me);
    RAG_REQUIRE((d_k_start == nullptr) == (d_k_len == nullptr), RAG_EINVAL, "%s: key starts and key lengths come together", me);
    if (n_seq == 0 || total_q == 0 || max_q_len == 0) return RAG_OK;
    RAG_REQUIRE(d_q && d_cu_q && d_out && ((d_k && d_v) || total_k == 0), RAG_EINVAL, "%s: null pointer", me);
    const int size = dtype == RAG_DTYPE_F32 ? 4 : 2;
    const auto off = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16; };
    RAG_REQUIRE(!off(d_q) && !off(d_k) && !off(d_v) && !off(d_out), RAG_EINVAL, "%s: pointers must be 16-byte aligned", me);
    RAG_REQUIRE(q_stride * size % 16 == 0 && k_row_stride * size % 16 == 0 && k_head_stride * size % 16 == 0 && v_row_stride * size % 16 == 0 &&
                v_head_stride * size % 16 == 0 && out_stride * size % 16 == 0, RAG_EINVAL, "%s: strides must be multiples of 16 bytes", me);
    RAG_REQUIRE(q_stride >= (int64_t)n_q_heads * head_dim && out_stride >= (int64_t)n_q_heads * head_dim, RAG_EINVAL,
                "%s: a row's stride is smaller than the row", me);
    RAG_REQUIRE(k_row_stride >= 0 && v_row_stride >= 0 && k_row_stride <= (1 << 25) / size && v_row_stride <= (1 << 25) / size, RAG_ELIMIT,
                "%s: rows of keys and values lie at most 32 MB apart", me);
    RAG_REQUIRE(workspace_bytes >= 0, RAG_EINVAL, "%s: bad workspace", me);
    WinArgs a;
    a.q = d_q; a.k = d_k; a.v = d_v; a.out = d_out; a.cu_q = d_cu_q; a.k_start = d_k_start; a.k_len = d_k_len;
    a.q_stride = q_stride; a.k_row = k_row_stride; a.k_head = k_head_stride; a.v_row = v_row_stride; a.v_head = v_head_stride;
    a.out_stride = out_stride; a.total_q = total_q; a.total_k = total_k;
    a.n_seq = n_seq; a.max_q = max_q_len; a.max_k = d_k_start ? max_k_len : max_q_len; a.hq = n_q_heads; a.hkv = n_kv_heads;
    a.left = window_left >= FAR ? -1 : window_left;
    a.right = window_right >= FAR ? -1 : window_right;
    a.sinks = n_sinks;
    a.scale = scale * 1.4426950408889634f;
    RAG_REQUIRE(!off(d_workspace) && (d_workspace || workspace_bytes == 0), RAG_EINVAL, "%s: bad workspace", me);
    hipStream_t stream = (hipStream_t)stream_;
    if (dtype == RAG_DTYPE_F32) return window_by_dim<float>(a, head_dim, d_workspace, workspace_bytes, stream);
    if (dtype == RAG_DTYPE_BF16) return window_by_dim<bf16>(a, head_dim, d_workspace, workspace_bytes, stream);
    return window_by_dim<f16>(a, head_dim, d_workspace, workspace_bytes, stream);
}
