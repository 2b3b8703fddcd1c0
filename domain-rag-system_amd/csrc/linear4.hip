// Products of a few rows with 4-bit weights: y[m][n] = sum_k x[m][k] w[n][k] + bias[n],
// w[n][k] = scale[n][k / G] * code[n][k] + offset[n][k / G] (no offsets: scale * (code - 8)).  The dense layers of an
// encoder for one query's tokens (MedicalEmbedder.encode of one text, reference src/indexing/embedder.py:65-71), where
// reading the weights is what the layer costs.  gfx950 only.
#include "common.h"

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
};

// The eight codes of a 32-bit word as eight 16-bit floats 16 + code: the code lands in the top mantissa bits of 16.0, so
// a pair costs one shift and one and-or, and no conversion.  Slots 0..7 hold the codes 0 4 1 5 2 6 3 7.
template <typename E> struct Code16;
template <> struct Code16<bf16> {
    typedef bf16x8 x8;
    static constexpr uint32_t MASK = 0x00780078u, BASE = 0x41804180u, ONES = 0x3f803f80u;
    __device__ static f32x4 mfma(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    __device__ static uint4 unpack(uint32_t w) {
        return make_uint4((w << 3 & MASK) | BASE, (w >> 1 & MASK) | BASE, (w >> 5 & MASK) | BASE, (w >> 9 & MASK) | BASE);
    }
};
template <> struct Code16<f16> {
    typedef f16x8 x8;
    static constexpr uint32_t MASK = 0x03c003c0u, BASE = 0x4c004c00u, ONES = 0x3c003c00u;
    __device__ static f32x4 mfma(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    __device__ static uint4 unpack(uint32_t w) {
        return make_uint4((w << 6 & MASK) | BASE, (w << 2 & MASK) | BASE, (w >> 2 & MASK) | BASE, (w >> 6 & MASK) | BASE);
    }
};

// Eight neighbouring values of a row of x as matrix operands in the order of the codes.  16-bit x is one operand; fp32 x
// is cut into three bf16 pieces of 8 significant bits each (exact: x = p0 + p1 + p2), three products with fp32 sums.
template <typename T> struct XFrag {
    typedef T E;
    static constexpr int PARTS = 1;
    uint4 v;
    __device__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
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

// A workgroup takes 16 rows of the weights and 16 * MT rows of x; its waves take the 128-column blocks of the weights in
// turn and add their sums up through LDS.  x is the A operand of v_mfma_f32_16x16x32, the codes are the B operand, so a lane
// ends with its own weight row's sums for four rows of x, and a group's scale is one value per lane.
//
// Lane (r, q) loads 16 bytes of row r, the codes of columns 32 q .. 32 q + 31 (64 contiguous bytes a row and load); a 4 x 4
// transposition of words between the four lanes of a row (four cross-row swaps) turns them into the operands of four
// steps of 32 columns, columns 8 q .. 8 q + 7 each, so that a step never mixes two groups and the weights need no layout
// of their own in memory.
//
// The operand holds 16 + code.  With c = sum x (16 + code) and X = sum x over a group (the same product with ones),
// sum x w = scale c + (offset - 16 scale) X.
template <typename T, int MT, int GROUP>
__global__ __launch_bounds__(1024) void linear4_kernel(Lin4Args a) {
    typedef XFrag<T> XF;
    typedef typename XF::E E;
    typedef Code16<E> C16;
    typedef typename C16::x8 x8;
    constexpr int NG = 128 / GROUP;                          // groups of a block
    constexpr int SPG = GROUP / 32;                          // steps of a group
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = (int)(blockDim.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int row = min((int)blockIdx.x * 16 + r, a.n - 1);  // (rows beyond the last repeat it and are not stored)
    const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
    const int groups = a.k / GROUP, blocks = (a.k + 127) / 128;
    const uint8_t* codes = a.codes + (int64_t)row * (a.k / 2);
    const T* scales = reinterpret_cast<const T*>(a.scales) + (int64_t)row * groups;
    const T* offsets = a.offsets ? reinterpret_cast<const T*>(a.offsets) + (int64_t)row * groups : nullptr;
    const T* x[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t] = reinterpret_cast<const T*>(a.x) + min(m0 + 16 * t + r, a.m - 1) * a.x_stride + 8 * q;

    struct Block { uint4 w; T s[NG], o[NG]; };
    auto load = [&](int blk, Block& b) {
        const int col = min(128 * blk + 32 * q, a.k - 32);   // (a piece beyond the row belongs to a step that is skipped)
        b.w = *reinterpret_cast<const uint4*>(codes + (col >> 1));
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int g = min(blk * NG + i, groups - 1);
            b.s[i] = scales[g];
            if (offsets) b.o[i] = offsets[g];
        }
    };
    f32x4 y[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) y[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const x8 ones = __builtin_bit_cast(x8, make_uint4(C16::ONES, C16::ONES, C16::ONES, C16::ONES));

    Block cur;
    if (wave < blocks) load(wave, cur);
    for (int blk = wave; blk < blocks; blk += waves) {
        Block next;
        if (blk + waves < blocks) load(blk + waves, next);
        uint32_t w[4] = {cur.w.x, cur.w.y, cur.w.z, cur.w.w};
        {
            auto p = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
            w[0] = p[0]; w[2] = p[1];
            p = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
            w[1] = p[0]; w[3] = p[1];
            p = __builtin_amdgcn_permlane16_swap(w[0], w[1], false, false);
            w[0] = p[0]; w[1] = p[1];
            p = __builtin_amdgcn_permlane16_swap(w[2], w[3], false, false);
            w[2] = p[0]; w[3] = p[1];
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            if (blk * 128 + g * GROUP >= a.k) break;         // (k is a whole number of groups)
            const float s = (float)cur.s[g];
            const float off = (offsets ? (float)cur.o[g] : -8.f * s) - 16.f * s;
            f32x4 c[MT], X[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) c[t] = X[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < SPG; ++i) {
                const int step = g * SPG + i;
                const x8 code = __builtin_bit_cast(x8, C16::unpack(w[step]));
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    XF xf;
                    xf.load(x[t] + 128 * blk + 32 * step);
                    uint4 part[XF::PARTS];
                    xf.parts(part);
#pragma unroll
                    for (int p = 0; p < XF::PARTS; ++p) {
                        const x8 xa = __builtin_bit_cast(x8, part[p]);
                        c[t] = C16::mfma(xa, code, c[t]);
                        X[t] = C16::mfma(xa, ones, X[t]);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) y[t][i] = fmaf(s, c[t][i], fmaf(off, X[t][i], y[t][i]));
        }
        cur = next;
    }

    // the waves' sums, in the order of the waves
    f32x4* part = reinterpret_cast<f32x4*>(smem);            // [waves][MT][64]
#pragma unroll
    for (int t = 0; t < MT; ++t) part[(wave * MT + t) * 64 + lane] = y[t];
    __syncthreads();
    for (int i = tid; i < MT * 64; i += (int)blockDim.x) {
        f32x4 sum = part[i];
        for (int v = 1; v < waves; ++v) sum += part[v * MT * 64 + i];
        const int n = (int)blockIdx.x * 16 + (i & 15);
        const int64_t m = m0 + 16 * (i >> 6) + 4 * ((i & 63) >> 4);
        if (n >= a.n) continue;
        const float bias = a.bias ? (float)reinterpret_cast<const T*>(a.bias)[n] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (m + j < a.m) reinterpret_cast<T*>(a.y)[(m + j) * a.y_stride + n] = (T)(sum[j] + bias);
    }
}

template <typename T, int MT>
int linear4_by_group(const Lin4Args& a, hipStream_t stream) {
    const int tiles = (a.n + 15) / 16, blocks = (a.k + 127) / 128;
    const int64_t my = ceil_div64(a.m, 16 * MT);
    RAG_REQUIRE(my <= 65535, RAG_ELIMIT, "rag_enc_linear4: too many rows of x");
    int waves = 4;
    while (waves < 16 && waves < blocks && (int64_t)tiles * my * waves < 4096) waves *= 2;
    const dim3 grid((unsigned)tiles, (unsigned)my);
    const size_t lds = (size_t)waves * MT * 1024;
    if (a.group == 32) linear4_kernel<T, MT, 32><<<grid, 64 * waves, lds, stream>>>(a);
    else if (a.group == 64) linear4_kernel<T, MT, 64><<<grid, 64 * waves, lds, stream>>>(a);
    else linear4_kernel<T, MT, 128><<<grid, 64 * waves, lds, stream>>>(a);
    RAG_HIP_TRY(hipGetLastError());
    return RAG_OK;
}

template <typename T>
int linear4_launch(const Lin4Args& a, hipStream_t stream) {
    if (a.m <= 16) return linear4_by_group<T, 1>(a, stream);
    if (a.m <= 32) return linear4_by_group<T, 2>(a, stream);
    return linear4_by_group<T, 4>(a, stream);
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
    RAG_REQUIRE(m < (1ll << 31) && n < (1 << 30) && k < (1 << 30), RAG_ELIMIT, "%s: sizes beyond the limit", me);
    if (m == 0) return RAG_OK;
    RAG_REQUIRE(d_x && d_codes && d_scales && d_y, RAG_EINVAL, "%s: null pointer", me);
    const int size = dtype == RAG_DTYPE_F32 ? 4 : 2;
    RAG_REQUIRE(reinterpret_cast<uintptr_t>(d_x) % 16 == 0 && reinterpret_cast<uintptr_t>(d_codes) % 16 == 0 && x_stride * size % 16 == 0,
                RAG_EINVAL, "%s: x, its rows and the codes must be 16-byte aligned", me);
    RAG_REQUIRE(reinterpret_cast<uintptr_t>(d_scales) % size == 0 && reinterpret_cast<uintptr_t>(d_offsets) % size == 0 &&
                reinterpret_cast<uintptr_t>(d_bias) % size == 0 && reinterpret_cast<uintptr_t>(d_y) % size == 0, RAG_EINVAL,
                "%s: misaligned pointer", me);
    RAG_REQUIRE((m == 1 || x_stride >= k) && (m == 1 || y_stride >= n), RAG_EINVAL, "%s: a row's stride is smaller than the row", me);
    Lin4Args a{d_x, d_codes, d_scales, d_offsets, d_bias, d_y, x_stride, y_stride, m, n, k, group};
    hipStream_t stream = (hipStream_t)stream_;
    if (dtype == RAG_DTYPE_F32) return linear4_launch<float>(a, stream);
    if (dtype == RAG_DTYPE_BF16) return linear4_launch<bf16>(a, stream);
    return linear4_launch<f16>(a, stream);
}
