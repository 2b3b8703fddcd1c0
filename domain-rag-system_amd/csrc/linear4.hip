// Products of a few rows with 4-bit weights: y[m][n] = sum_k x[m][k] w[n][k] + bias[n],
// w[n][k] = scale[n][k / G] * code[n][k] + offset[n][k / G] (no offsets: scale * (code - 8)).  The dense layers of an
// encoder for one query's tokens, where reading the weights is what the layer costs (beside the 16-bit and fp32 layers of
// MedicalEmbedder's encoders, reference src/indexing/embedder.py:65-71).  gfx950 only.
// Measured, bf16, group 32, n 16383, k 8192 (75 MB): one token 20.7 us (3.6 TB/s; a large copy moves 4.7), 13 tokens 24 (147
// TFLOP/s of products: the codes are unpacked by the vector units beside them, and the waves meet once per workgroup), 64
// tokens 54; n 4096, k 4096, group 128 (8.9 MB): 5.3, 6.2 and 10.
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));

struct Lin4Args {
    const void* x;
    const uint8_t* codes;
    const void *scales, *offsets, *bias;
    void* y;
    int64_t x_stride, y_stride, m;
    int32_t n, k, group;
    int32_t image;                   // where the images of x begin in LDS
    int32_t chunk;                   // 128-column blocks whose scales are in LDS at a time
};

// The eight codes of a 32-bit word as eight 16-bit floats 16 + code: the code lands in the top mantissa bits of 16.0, so
// a pair costs one shift and one and-or, and no conversion.  Slots 0..7 hold the codes 0 4 1 5 2 6 3 7.
template <typename E> struct Code16;
template <> struct Code16<bf16> {
    typedef bf16x8 x8;
    static constexpr uint32_t MASK = 0x00780078u, BASE = 0x41804180u, ONES = 0x3f803f80u;
    __device__ static f32x4 mfma(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    __device__ static uint4 unpack(uint32_t w, uint32_t mask, uint32_t base) {
        return make_uint4((w << 3 & mask) | base, (w >> 1 & mask) | base, (w >> 5 & mask) | base, (w >> 9 & mask) | base);
    }
};
template <> struct Code16<f16> {
    typedef f16x8 x8;
    static constexpr uint32_t MASK = 0x03c003c0u, BASE = 0x4c004c00u, ONES = 0x3c003c00u;
    __device__ static f32x4 mfma(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    __device__ static uint4 unpack(uint32_t w, uint32_t mask, uint32_t base) {
        return make_uint4((w << 6 & mask) | base, (w << 2 & mask) | base, (w >> 2 & mask) | base, (w >> 6 & mask) | base);
    }
};

// Eight neighbouring values of a row of x as matrix operands in the order of the codes.  16-bit x is one operand; fp32 x
// is cut into three bf16 pieces of 8 significant bits each (exact: x = p0 + p1 + p2), three products with fp32 sums.
template <typename T> struct XFrag {
    typedef T E;
    static constexpr int PARTS = 1;
    uint4 v;
    __device__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
    // columns 8 piece .. of a row of an image in LDS whose 16-byte pieces lie at p ^ s
    __device__ void load(const unsigned char* row, int piece, int s) { v = *reinterpret_cast<const uint4*>(row + (piece ^ s) * 16); }
    __device__ void parts(uint4* out) const {
        out[0].x = __builtin_amdgcn_perm(v.z, v.x, 0x05040100u);
        out[0].y = __builtin_amdgcn_perm(v.z, v.x, 0x07060302u);
        out[0].z = __builtin_amdgcn_perm(v.w, v.y, 0x05040100u);
        out[0].w = __builtin_amdgcn_perm(v.w, v.y, 0x07060302u);
    }
};
template <> struct XFrag<float> {
    typedef bf16 E;
    static constexpr int PARTS = 3;
    float4 a, b;
    __device__ void load(const float* p) {
        a = *reinterpret_cast<const float4*>(p);
        b = *reinterpret_cast<const float4*>(p + 4);
    }
    __device__ void load(const unsigned char* row, int piece, int s) {
        a = *reinterpret_cast<const float4*>(row + ((2 * piece) ^ s) * 16);
        b = *reinterpret_cast<const float4*>(row + ((2 * piece + 1) ^ s) * 16);
    }
    __device__ static void cut(float lo, float hi, uint32_t* out) {
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const uint32_t l = __float_as_uint(lo), h = __float_as_uint(hi);
            out[i] = __builtin_amdgcn_perm(h, l, 0x07060302u);
            lo -= __uint_as_float(l & 0xffff0000u);
            hi -= __uint_as_float(h & 0xffff0000u);
        }
    }
    __device__ void parts(uint4* out) const {
        uint32_t w[4][3];
        cut(a.x, b.x, w[0]);
        cut(a.y, b.y, w[1]);
        cut(a.z, b.z, w[2]);
        cut(a.w, b.w, w[3]);
#pragma unroll
        for (int i = 0; i < 3; ++i) out[i] = make_uint4(w[0][i], w[1][i], w[2][i], w[3][i]);
    }
};

// The most waves an instance is compiled for: 1024 threads leave 128 registers a lane, enough for one row tile and 16-bit x, and for
// two with x as operands; with x by rows 3 to 13 registers of two row tiles go to scratch, in launches of fewer waves too
template <typename T, int RT> constexpr int max_waves() { return RT <= 2 && sizeof(T) == 2 ? 16 : 8; }

// A group's scale and offset as one value
template <typename T> struct ScalePair {
    typedef uint32_t type;
    __device__ static type make(T s, T o) {
        return (uint32_t)__builtin_bit_cast(uint16_t, s) | (uint32_t)__builtin_bit_cast(uint16_t, o) << 16;
    }
    __device__ static void split(type p, float& s, float& o) {
        s = (float)__builtin_bit_cast(T, (uint16_t)p);
        o = (float)__builtin_bit_cast(T, (uint16_t)(p >> 16));
    }
};
template <> struct ScalePair<float> {
    typedef float2 type;
    __device__ static type make(float s, float o) { return make_float2(s, o); }
    __device__ static void split(type p, float& s, float& o) { s = p.x; o = p.y; }
};

// The sums of x times 16 + code, and 16 scales, can leave the range of fp32 (x of 1e35 and more, scales of 1e37) where x times
// whole weights does not.  So what is not finite is computed again from those, by a wave: finite_row tells whether x itself
// is the reason, which leaves the value as it is (n 16384, k 8192, bf16: 13 rows, a NaN in one of them, 28 us; 64 rows with a NaN each
// 220, without 43).  With neither, the look at the sums costs 0.1 us.
template <typename T>
__device__ bool finite_row(const Lin4Args& a, int64_t m, int lane) {
    const T* x = reinterpret_cast<const T*>(a.x) + m * a.x_stride;
    struct alignas(16) Piece { T v[8]; };
    for (int c = 8 * lane; __any(c < a.k); c += 512) {       // (rows are whole pieces)
        bool good = true;
        if (c < a.k) {
            const Piece p = *reinterpret_cast<const Piece*>(x + c);
#pragma unroll
            for (int e = 0; e < 8; ++e) good &= isfinite((float)p.v[e]);
        }
        if (!__all(good)) return false;
    }
    return true;
}
template <typename T>
__device__ float whole_product(const Lin4Args& a, int64_t m, int64_t n, int lane) {
    const T* x = reinterpret_cast<const T*>(a.x) + m * a.x_stride;
    const uint8_t* codes = a.codes + n * (a.k / 2);
    const T* scales = reinterpret_cast<const T*>(a.scales) + n * (a.k / a.group);
    const T* offsets = reinterpret_cast<const T*>(a.offsets) + n * (a.k / a.group);
    float sum = 0.f;
    for (int c = 8 * lane; c < a.k; c += 512) {              // (eight columns never cross a group)
        const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + c / 2);
        const float s = (float)scales[c / a.group], o = a.offsets != nullptr ? (float)offsets[c / a.group] : 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float code = (float)(w >> (4 * e) & 15u);
            sum = fmaf((float)x[c + e], a.offsets != nullptr ? fmaf(s, code, o) : s * (code - 8.f), sum);
        }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
    return sum;
}

// A workgroup takes 16 * RT rows of the weights and 16 * MT rows of x; its waves take the 128-column blocks of the weights
// in turn and add their sums up through LDS.  x is the A operand of v_mfma_f32_16x16x32, the codes are the B operand, so a
// lane ends with its own weight row's sums for four rows of x, and a group's scale is one value per lane.
//
// Lane (r, q) loads 16 bytes of row r, the codes of columns 32 q .. 32 q + 31 (64 contiguous bytes a row and load); a 4 x 4
// transposition of words between the four lanes of a row (four cross-row swaps) turns them into the operands of four
// steps of 32 columns, columns 8 q .. 8 q + 7 each, so that a step never mixes two groups and the weights need no layout
// of their own in memory.
//
// Scales and offsets go through LDS, a chunk of blocks at a time, read from memory row by row: loaded by the lane that needs
// them they are 16 cache lines a load for 2 bytes of each, which the L1 has lost again when the next group's are read (measured at
// n 16384, k 8192, group 64, m 1: codes alone 12.7 us, with scales loaded by lane 26.7 us).
//
// The operand holds 16 + code.  With c = sum x (16 + code) and X = sum x over a group (the same product with ones),
// sum x w = scale c + (offset - 16 scale) X.  These sums are some five times larger than what is left of them (fp32 x: error 4e-7
// of the result's size, with whole weights 2e-7), and may overflow where it does not: see whole_product.
//
// The loads of the wave's next block are issued before the products of this one.  Loads return in order: x, which comes from the L2, is
// asked for before the codes of the next block, which come from memory, or with its own block (MT == 1).
// x is loaded as the operands lie (16 rows, 64 bytes of each a load), or with ROWS in whole pieces of few rows, which go
// through an image in LDS: rows of x lie a power of two apart as a rule, so that 16 of them meet on one channel of the L2.
template <typename T, int MT, int RT, int GROUP, bool ROWS>
__global__ __launch_bounds__((64 * max_waves<T, RT>())) void linear4_kernel(Lin4Args a) {
    typedef XFrag<T> XF;
    typedef typename XF::E E;
    typedef Code16<E> C16;
    typedef typename C16::x8 x8;
    constexpr int NG = 128 / GROUP;                          // groups of a block
    constexpr int SPG = GROUP / 32;                          // steps of a group
    constexpr int RUN = sizeof(T) == 4 ? 1 : SPG;            // steps summed before the scale: c, five times the size of what is left of it, is
                                                             // kept short where its last bits count (group 128: error 8e-7, a step 5e-7)
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, waves = (int)(blockDim.x >> 6);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
    const int groups = a.k / GROUP, full = a.k / 128;        // blocks that k fills
    const bool has_off = a.offsets != nullptr;
    const float s_mul = has_off ? -16.f : -24.f, o_mul = has_off ? 1.f : 0.f;
    // byte offsets of the lane's rows from the first row of the workgroup (k < 2^26: they fit 32 bits)
    const int64_t row0 = (int64_t)blockIdx.x * (16 * RT);
    const uint8_t* codes = a.codes + row0 * (a.k / 2);
    const T* scales = reinterpret_cast<const T*>(a.scales) + row0 * groups;
    const T* offsets = has_off ? reinterpret_cast<const T*>(a.offsets) + row0 * groups : scales;
    const int rows_here = (int)min((int64_t)(16 * RT), a.n - row0);
    uint32_t code_at[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        code_at[t] = (uint32_t)min(16 * t + r, rows_here - 1) * (uint32_t)(a.k / 2) + 16 * q;    // (rows beyond the last repeat it and are not stored)
    }
    constexpr int X_ROWB = 128 * (int)sizeof(T), X_PIECES = X_ROWB / 16, X_ROWS = 1024 / X_ROWB, X_LOADS = MT * X_ROWB / 64;
    const uint8_t* xbase = reinterpret_cast<const uint8_t*>(a.x) + m0 * a.x_stride * (int64_t)sizeof(T);
    const int m_here = (int)min((int64_t)(16 * MT), a.m - m0);
    uint32_t x_at[X_LOADS];                                  // ROWS: the lane's rows of x, in bytes (they fit by the limit on the stride)
#pragma unroll
    for (int i = 0; i < X_LOADS; ++i)
        x_at[i] = (uint32_t)min(i * X_ROWS + lane / X_PIECES, m_here - 1) * (uint32_t)(a.x_stride * (int64_t)sizeof(T));
    unsigned char* image = smem + a.image + wave * (16 * MT * X_ROWB);
    const T* x[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t] = reinterpret_cast<const T*>(a.x) + min(m0 + 16 * t + r, a.m - 1) * a.x_stride + 8 * q;

    struct Block { uint4 w[RT]; };
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    struct XRows { u32x4 raw[X_LOADS]; };
    struct XFrags { XF f[4][MT]; };
    typedef typename std::conditional<ROWS, XRows, XFrags>::type XBlock;
    auto load = [&](int blk, Block& b) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            b.w[t] = *reinterpret_cast<const uint4*>(codes + (code_at[t] + (uint32_t)blk * 64));
        }
    };
    auto load_x = [&](int blk, XBlock& b) {
        if constexpr (ROWS) {
            const int last = min(128, a.k - 128 * blk) * (int)sizeof(T) / 16 - 1;         // (in a row's last block: pieces beyond it repeat it)
#pragma unroll
            for (int i = 0; i < X_LOADS; ++i)
                b.raw[i] = *reinterpret_cast<const u32x4*>(xbase + (int64_t)blk * X_ROWB + (x_at[i] + 16 * min(lane % X_PIECES, last)));
        } else {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const T* p = x[t] + 128 * blk;
#pragma unroll
                for (int i = 0; i < 4; ++i) b.f[i][t].load(p + 32 * i);
            }
        }
    };
    f32x4 y[RT][MT];
#pragma unroll
    for (int u = 0; u < RT; ++u)
#pragma unroll
        for (int t = 0; t < MT; ++t) y[u][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const x8 ones = __builtin_bit_cast(x8, make_uint4(C16::ONES, C16::ONES, C16::ONES, C16::ONES));
    // one constant in a vector, one in a scalar register: the and-or of a pair of codes is then one instruction
    uint32_t mask = C16::MASK, base = C16::BASE;
    asm("" : "+v"(mask));
    asm("" : "+s"(base));

    // [16 * RT rows][groups of the chunk], scale and offset side by side; an odd row stride spreads the 16 rows over the banks
    typedef typename ScalePair<T>::type Pair;
    Pair* pairs = reinterpret_cast<Pair*>(smem);
    const int pair_stride = (a.chunk * NG) | 1;
    // g0: the block's first group in the chunk
    auto process = [&](const Block& cur, const XBlock& xcur, int g0, int steps) {
        if constexpr (ROWS) {                                // (LDS accesses of a wave stay in order)
#pragma unroll
            for (int i = 0; i < X_LOADS; ++i) {
                const int row = i * X_ROWS + lane / X_PIECES;
                *reinterpret_cast<u32x4*>(image + row * X_ROWB + ((lane % X_PIECES) ^ (row & 15)) * 16) = xcur.raw[i];
            }
            __builtin_amdgcn_wave_barrier();
        }
        uint32_t w[RT][4];
#pragma unroll
        for (int u = 0; u < RT; ++u) {
            auto p = __builtin_amdgcn_permlane32_swap(cur.w[u].x, cur.w[u].z, false, false);
            w[u][0] = p[0]; w[u][2] = p[1];
            p = __builtin_amdgcn_permlane32_swap(cur.w[u].y, cur.w[u].w, false, false);
            w[u][1] = p[0]; w[u][3] = p[1];
            p = __builtin_amdgcn_permlane16_swap(w[u][0], w[u][1], false, false);
            w[u][0] = p[0]; w[u][1] = p[1];
            p = __builtin_amdgcn_permlane16_swap(w[u][2], w[u][3], false, false);
            w[u][2] = p[0]; w[u][3] = p[1];
        }
#pragma unroll
        for (int step0 = 0; step0 < 4; step0 += RUN) {
            if (step0 >= steps) break;                       // (k is a whole number of groups)
            f32x4 c[RT][MT], X[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                X[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < RT; ++u) c[u][t] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int step = step0; step < step0 + RUN; ++step) {
                x8 code[RT];
#pragma unroll
                for (int u = 0; u < RT; ++u) code[u] = __builtin_bit_cast(x8, C16::unpack(w[u][step], mask, base));
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    uint4 part[XF::PARTS];
                    if constexpr (ROWS) {
                        XF xf;
                        xf.load(image + (16 * t + r) * X_ROWB, 4 * step + q, r);
                        xf.parts(part);
                    } else {
                        xcur.f[step][t].parts(part);
                    }
#pragma unroll
                    for (int p = 0; p < XF::PARTS; ++p) {
                        const x8 xa = __builtin_bit_cast(x8, part[p]);
                        X[t] = C16::mfma(xa, ones, X[t]);
#pragma unroll
                        for (int u = 0; u < RT; ++u) c[u][t] = C16::mfma(xa, code[u], c[u][t]);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < RT; ++u) {
                float s, off;
                ScalePair<T>::split(pairs[(16 * u + r) * pair_stride + g0 + step0 / SPG], s, off);
                off = fmaf(s_mul, s, off * o_mul);
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[u][t][i] = fmaf(s, c[u][t][i], fmaf(off, X[t][i], y[u][t][i]));
            }
        }
    };

    for (int c0 = 0; c0 * 128 < a.k; c0 += a.chunk) {
        const int c_full = min(full, c0 + a.chunk);           // whole blocks [c0, c_full)
        // a wave's blocks are neighbours: the two that share the 128-byte lines of a row follow each other
        const int per = (c_full - c0 + waves - 1) / waves;
        const int first = c0 + wave * per, last = min(c_full, first + per) - 1;
        Block b0, b1;
        XBlock x0, x1;
        if (first <= last) {
            if (MT == 1) load_x(first, x0);
            load(first, b0);
        }
        {
            const int g_first = c0 * NG, g_n = min(groups - g_first, a.chunk * NG);
            const int total = rows_here * g_n;
            for (int i = tid; i < total; i += 4 * (int)blockDim.x) {
                T sv[4], ov[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int e = min(i + j * (int)blockDim.x, total - 1), row = e / g_n;
                    const uint32_t at = (uint32_t)row * (uint32_t)groups + (uint32_t)(g_first + e - row * g_n);
                    sv[j] = scales[at];
                    ov[j] = offsets[at];
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int e = min(i + j * (int)blockDim.x, total - 1), row = e / g_n;
                    pairs[row * pair_stride + e - row * g_n] = ScalePair<T>::make(sv[j], ov[j]);
                }
            }
        }
        __syncthreads();
        for (int blk = first; blk <= last; blk += 2) {
            const int second = min(blk + 1, last), third = min(blk + 2, last);
            if (MT == 1) load_x(second, x1);
            else load_x(blk, x0);
            __builtin_amdgcn_sched_barrier(0);
            load(second, b1);
            __builtin_amdgcn_sched_barrier(0);
            process(b0, x0, (blk - c0) * NG, 4);
            if (blk == last) break;
            if (MT == 1) load_x(third, x0);
            else load_x(second, x1);
            __builtin_amdgcn_sched_barrier(0);
            load(third, b0);
            __builtin_amdgcn_sched_barrier(0);
            process(b1, x1, (second - c0) * NG, 4);
        }
        // the last block of a row that ends inside it, by the last wave: pieces beyond the row are loaded from its last 32
        // columns and belong to steps that are not taken
        if (a.k % 128 != 0 && full < c0 + a.chunk && wave == waves - 1) {
            const int col = min(128 * full + 32 * q, a.k - 32);
#pragma unroll
            for (int t = 0; t < RT; ++t) b0.w[t] = *reinterpret_cast<const uint4*>(codes + (code_at[t] - 16 * q + (uint32_t)(col >> 1)));
            if constexpr (ROWS) {
                load_x(full, x0);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int t = 0; t < MT; ++t) x0.f[i][t].load(x[t] + min(128 * full + 32 * i, a.k - 32));
            }
            process(b0, x0, (full - c0) * NG, (a.k % 128) / 32);
        }
        __syncthreads();                                     // the scales are read: the next chunk's, or the sums, go there
    }

    // the waves' sums, in the order of the waves
    f32x4* part = reinterpret_cast<f32x4*>(smem);            // [waves][RT][MT][64]
#pragma unroll
    for (int u = 0; u < RT; ++u)
#pragma unroll
        for (int t = 0; t < MT; ++t) part[((wave * RT + u) * MT + t) * 64 + lane] = y[u][t];
    __syncthreads();
    for (int i = tid; i < RT * MT * 64; i += (int)blockDim.x) {
        f32x4 sum = part[i];
        for (int v = 1; v < waves; ++v) sum += part[v * RT * MT * 64 + i];
        const int n0 = ((int)blockIdx.x * RT + i / (MT * 64)) * 16, n = n0 + (i & 15);
        const int64_t m1 = m0 + 16 * ((i / 64) % MT), m = m1 + 4 * ((i & 63) >> 4);
        const f32x4 none = sum - sum;                        // (0 where finite; the lanes of a wave are at the same n0 and m1)
        const bool bad = !(none[0] + none[1] + none[2] + none[3] == 0.f) && n < a.n;
        if (__builtin_expect(__any(bad), 0)) {
#pragma unroll 1
            for (int row = 0; row < 16 && m1 + row < a.m; ++row) {
                float mine = sum[0];
#pragma unroll
                for (int j = 1; j < 4; ++j) mine = (row & 3) == j ? sum[j] : mine;
                uint64_t rest = __ballot(bad && lane >> 4 == row >> 2 && !isfinite(mine));
                if (rest == 0 || !finite_row<T>(a, m1 + row, lane)) continue;
                for (; rest != 0; rest &= rest - 1) {
                    const int from = __builtin_ctzll(rest);
                    const float again = whole_product<T>(a, m1 + row, n0 + (from & 15), lane);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (lane == from && (row & 3) == j) sum[j] = again;
                }
            }
        }
        if (n >= a.n) continue;
        const float bias = a.bias ? (float)reinterpret_cast<const T*>(a.bias)[n] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (m + j < a.m) reinterpret_cast<T*>(a.y)[(m + j) * a.y_stride + n] = (T)(sum[j] + bias);
    }
}

template <typename T, int MT, int RT, bool ROWS>
int linear4_by_group(Lin4Args a, hipStream_t stream) {
    const int tiles = (a.n + 16 * RT - 1) / (16 * RT), blocks = (a.k + 127) / 128;
    const int64_t my = ceil_div64(a.m, 16 * MT);
    RAG_REQUIRE(my <= 65535, RAG_ELIMIT, "rag_enc_linear4: too many rows of x");
    int waves = 4;
    while (waves < max_waves<T, RT>() && waves < blocks && (int64_t)tiles * my * waves < 2048) waves *= 2;
    const dim3 grid((unsigned)tiles, (unsigned)my);
    // at most 32 KB of scales at a time (the images of x take at most 64)
    const int ng = 128 / a.group, row_bytes = 16 * RT * (int)sizeof(typename ScalePair<T>::type);
    const int images = ROWS ? waves * 16 * MT * 128 * (int)sizeof(T) : 0;
    a.chunk = std::min(blocks, 32768 / (row_bytes * ng));
    a.image = (row_bytes * ((a.chunk * ng) | 1) + 1023) / 1024 * 1024;
    const size_t lds = std::max((size_t)a.image + images, (size_t)waves * MT * RT * 1024);
#define RAG_LINEAR4_LAUNCH(G)                                                            \
    do {                                                                                 \
        RAG_GRANT_LDS((linear4_kernel<T, MT, RT, G, ROWS>), lds);                         \
        linear4_kernel<T, MT, RT, G, ROWS><<<grid, 64 * waves, lds, stream>>>(a);         \
    } while (0)
    if (a.group == 32) RAG_LINEAR4_LAUNCH(32);
    else if (a.group == 64) RAG_LINEAR4_LAUNCH(64);
    else RAG_LINEAR4_LAUNCH(128);
#undef RAG_LINEAR4_LAUNCH
    RAG_HIP_TRY(hipGetLastError());
    return RAG_OK;
}

// x by whole rows from 5 rows on (n 4096, k 4096: m 4 6.1 us as operands, 6.0 by rows, m 13 7.9 and 6.2); not where fp32
// rows and 64 rows of weights are more than the registers hold (n 16383, k 8192, m 24: 57 us, by rows 71).
template <typename T, int MT, int RT>
int linear4_tile(const Lin4Args& a, hipStream_t stream) {
    if constexpr (sizeof(T) == 2 && RT == 4) return linear4_by_group<T, MT, RT, true>(a, stream);       // (64 rows of weights: more than 16 of x)
    else if constexpr (RT == 4) return linear4_by_group<T, MT, RT, false>(a, stream);
    else return a.m > 4 ? linear4_by_group<T, MT, RT, true>(a, stream) : linear4_by_group<T, MT, RT, false>(a, stream);
}

// The smallest tile with which the workgroups are on the chip at once, one per compute unit: x is read by each of them, so
// fewer and larger ones read less, but a second round costs as much as the first (k 4096, group 128, x as operands: n 4096, m 16: 16 x 16
// tiles 10 us, 32 x 16 12; m 64: 16 x 16 23, 32 x 16 17, 64 x 16 13.2, and 16 x 64, 256 workgroups too, 19.9).  Beyond that the
// largest, up to 16 rows of x 32 x 16, which keep more waves on the chip for the weights (n 16383, k 8192: m 1 21 us, 64 x 16 26; m
// 13 23.8 and 26.9).
template <typename T>
int linear4_launch(const Lin4Args& a, hipStream_t stream) {
    const int64_t tiles = (a.n + 15) / 16, my = (a.m + 15) / 16;
    if (tiles * my <= 256) return linear4_tile<T, 1, 1>(a, stream);
    if (a.m <= 16 || (tiles + 1) / 2 * my <= 256) return linear4_tile<T, 1, 2>(a, stream);
    if ((tiles + 3) / 4 * my <= 256) return linear4_tile<T, 1, 4>(a, stream);
    return linear4_tile<T, 2, 4>(a, stream);
}

}  // namespace

extern "C" int rag_enc_linear4_dev(const void* d_x, int64_t x_stride, const uint8_t* d_codes, const void* d_scales,
                                   const void* d_offsets, const void* d_bias, int64_t m, int32_t n, int32_t k, int32_t group,
                                   int32_t dtype, void* d_y, int64_t y_stride, void* stream_) {
    const char* me = "rag_enc_linear4";
    RAG_REQUIRE(dtype == RAG_DTYPE_F32 || dtype == RAG_DTYPE_BF16 || dtype == RAG_DTYPE_F16, RAG_EINVAL, "%s: unknown dtype %d", me, dtype);
    RAG_REQUIRE(m >= 0 && n >= 1 && k >= 1, RAG_EINVAL, "%s: bad sizes", me);
    RAG_REQUIRE(group == 32 || group == 64 || group == 128, RAG_ELIMIT, "%s: the group must be 32, 64 or 128 (got %d)", me, group);
    RAG_REQUIRE(k % group == 0, RAG_ELIMIT, "%s: k = %d is not a multiple of the group %d", me, k, group);
    RAG_REQUIRE(m < (1ll << 31) && n < (1 << 28) && k < (1 << 26), RAG_ELIMIT, "%s: sizes beyond the limit", me);
    if (m == 0) return RAG_OK;
    RAG_REQUIRE(d_x && d_codes && d_scales && d_y, RAG_EINVAL, "%s: null pointer", me);
    const int size = dtype == RAG_DTYPE_F32 ? 4 : 2;
    RAG_REQUIRE(reinterpret_cast<uintptr_t>(d_x) % 16 == 0 && reinterpret_cast<uintptr_t>(d_codes) % 16 == 0 && x_stride * size % 16 == 0,
                RAG_EINVAL, "%s: x, its rows and the codes must be 16-byte aligned", me);
    RAG_REQUIRE(reinterpret_cast<uintptr_t>(d_scales) % size == 0 && reinterpret_cast<uintptr_t>(d_offsets) % size == 0 &&
                reinterpret_cast<uintptr_t>(d_bias) % size == 0 && reinterpret_cast<uintptr_t>(d_y) % size == 0, RAG_EINVAL,
                "%s: misaligned pointer", me);
    RAG_REQUIRE((m == 1 || x_stride >= k) && (m == 1 || y_stride >= n), RAG_EINVAL, "%s: a row's stride is smaller than the row", me);
    RAG_REQUIRE(m == 1 || x_stride <= (1 << 25) / size, RAG_ELIMIT, "%s: rows of x lie at most 32 MB apart", me);
    Lin4Args a{d_x, d_codes, d_scales, d_offsets, d_bias, d_y, x_stride, y_stride, m, n, k, group, 0, 0};
    hipStream_t stream = (hipStream_t)stream_;
    if (dtype == RAG_DTYPE_F32) return linear4_launch<float>(a, stream);
    if (dtype == RAG_DTYPE_BF16) return linear4_launch<bf16>(a, stream);
    return linear4_launch<f16>(a, stream);
}
