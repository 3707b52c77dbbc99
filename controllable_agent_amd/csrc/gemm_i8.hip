// Matrix product in 8-bit integers: y[m, n] = act( (sum_k a[m, k] w[n, k]) * sa[m] * sw[n] + bias[n] ), with a scale for each row of both
// operands, and the row quantiser that makes them: s = max|x| * fl(1/127), code = nearest whole number to fl(x / s) (ties to even).
//
// The sum is exact: |sum| <= K 128^2 < 2^31 up to K = 131071, the largest that the entry points take, whatever the order of the additions, so K may
// be split at will.  It is turned into a float once (24 bits) and scaled in single precision.
#include "common.h"
#include "host.h"

#include <atomic>

namespace fbhip {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));
// values side by side at any address: gfx950's global loads and stores need no alignment
typedef float floatx4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t uintx2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t uintx4_any __attribute__((ext_vector_type(4), aligned(2)));

constexpr int I8_BK = 128;                    // bytes of K in a step: one row of a tile is one 128-byte line

// ------------------------------------------------------------------------------------------------------------------ quantiser
__device__ __forceinline__ float i8_load(const void* x, size_t i, int type) {
    if (type == FBHIP_F32) return ((const float*)x)[i];
    const uint16_t h = ((const uint16_t*)x)[i];
    if (type == FBHIP_BF16) return __uint_as_float((uint32_t)h << 16);
    _Float16 f;
    __builtin_memcpy(&f, &h, 2);
    return (float)f;
}

// The largest magnitude is found on the bits, which order like the values; infinities and NaN come out above every number.
__device__ __forceinline__ uint32_t i8_top(uint32_t top, float x) { return max(top, __float_as_uint(x) & 0x7FFFFFFFu); }

// over groups of LANES lanes
template <int LANES>
__device__ __forceinline__ uint32_t i8_lanes_top(uint32_t top) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    return top;
}

struct I8Row { float scale, inv; bool zero, divide; };
// a row that holds a NaN or an infinity: the scale NaN and codes 0; a row of zeros, or one so small that its scale is 0: codes 0
__device__ __forceinline__ I8Row i8_row(uint32_t top) {
    I8Row r;
    const bool bad = top >= 0x7F800000u;
    r.scale = __uint_as_float(top) * (1.f / 127.f);       // (the reciprocal rounded to float32: within a step of the quotient)
    r.zero = bad || r.scale == 0.f;
    r.divide = r.scale < 0x1p-100f;                       // (the reciprocal would leave the range)
    r.inv = r.divide ? 1.f : __builtin_amdgcn_rcpf(r.scale);
    if (bad) r.scale = __uint_as_float(0x7FC00000u);
    return r;
}

// The codes of four values: x / s, rounded to float32 and then to the nearest whole number, ties to even.  x times the reciprocal is off by less than
// 5e-5 for |x / s| <= 127 (a step of v_rcp_f32, half a step of the product and of the quotient: 127 * 2.5 * 2^-23 = 3.8e-5), so that only where
// a value comes so near to a half the four are divided.  The conversion packs bytes of 0..255: 128 is added, and taken off in the top bits.
__device__ __forceinline__ uint32_t i8_codes(float a, float b, float c, float d, const I8Row& r) {
    const float x[4] = {a, b, c, d};
    float n[4], off = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float q = x[e] * r.inv;
        n[e] = rintf(q);
        off = fmaxf(off, fabsf(q - n[e]));
    }
    if (off >= 0.49995f || r.divide) {
#pragma unroll
        for (int e = 0; e < 4; ++e) n[e] = fminf(fmaxf(rintf(x[e] / r.scale), -127.f), 127.f);
    }
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) w = __builtin_amdgcn_cvt_pk_u8_f32(n[e] + 128.f, e, w);
    return r.zero ? 0u : w ^ 0x80808080u;
}

// values e of a 16-byte piece
template <bool WIDE>
__device__ __forceinline__ float i8_unpack(const uint32_t (&w)[4], int e, int type) {
    if (WIDE) return __uint_as_float(w[e & 3]);
    if (type == FBHIP_BF16) return __uint_as_float((e & 1) ? w[(e >> 1) & 3] & 0xFFFF0000u : w[(e >> 1) & 3] << 16);
    const uint16_t h = (uint16_t)(w[(e >> 1) & 3] >> (16 * (e & 1)));
    _Float16 g;
    __builtin_memcpy(&g, &h, 2);
    return (float)g;
}

// the piece at element k of a row of K: zero behind its end
template <bool WIDE>
__device__ __forceinline__ uint4 i8_piece(const char* base, int k, int K) {
    constexpr int V = WIDE ? 4 : 8;
    if (k + V <= K) {
        const uintx4_any w = *(const uintx4_any*)(base + (size_t)k * (16 / V));
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    for (int e = 0; e < K - k; ++e) {
        if (WIDE) w[e] = ((const uint32_t*)base)[k + e];
        else w[e >> 1] |= (uint32_t)((const uint16_t*)base)[k + e] << (16 * (e & 1));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Bound by memory: x is read once, the codes are written once (8192^2 bf16: 34 us, 6.0 TB/s, part of it from the Infinity Cache).
// A row in the registers of TPR threads: C pieces of 16 bytes a thread, read once, whatever the row's alignment.
template <int TPR, int C, bool WIDE>
__global__ void __launch_bounds__(256) quantize_rows_reg_kernel(const void* __restrict__ x, int64_t ldx, int type, int8_t* __restrict__ q, int64_t ldq,
                                                                float* __restrict__ scale, int rows, int K, int Kp) {
    constexpr int V = WIDE ? 4 : 8;                       // values of a piece (WIDE: fp32)
    __shared__ uint32_t red[4];
    const int t = threadIdx.x % TPR, row = blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    const bool live = row < rows;                         // (only TPR = 64 has rows behind the end)
    const char* base = (const char*)x + (size_t)(live ? row : rows - 1) * ldx * (16 / V);
    float v[C][V];
    uint32_t top = 0;
    uint4 raw[C];
#pragma unroll
    for (int c = 0; c < C; ++c) raw[c] = i8_piece<WIDE>(base, (c * TPR + t) * V, K);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
        for (int e = 0; e < V; ++e) {
            v[c][e] = i8_unpack<WIDE>(w, e, type);
            top = i8_top(top, v[c][e]);
        }
    }
    top = i8_lanes_top<64>(top);
    if (TPR == 256) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
        __syncthreads();
        top = max(max(red[0], red[1]), max(red[2], red[3]));
    }
    const I8Row r = i8_row(top);
    if (!live) return;
    int8_t* out = q + (size_t)row * ldq;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int k = (c * TPR + t) * V;
        if (k >= Kp) break;
        const uint32_t first = i8_codes(v[c][0], v[c][1], v[c][2], v[c][3], r);          // (zeros behind K stay zeros)
        if (WIDE) *(uint32_t*)(out + k) = first;
        else *(uint2*)(out + k) = make_uint2(first, i8_codes(v[c][V - 4], v[c][V - 3], v[c][V - 2], v[c][V - 1], r));
    }
    if (t == 0) scale[row] = r.scale;
}

// Longer rows: a workgroup reads them twice.
__global__ void __launch_bounds__(256) quantize_rows_kernel(const void* __restrict__ x, int64_t ldx, int type, int8_t* __restrict__ q, int64_t ldq,
                                                            float* __restrict__ scale, int K, int Kp) {
    __shared__ uint32_t red[4];
    const int tid = threadIdx.x;
    const size_t base = (size_t)blockIdx.x * ldx;
    uint32_t top = 0;
    for (int k = tid; k < K; k += 256) top = i8_top(top, i8_load(x, base + k, type));
    top = i8_lanes_top<64>(top);
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
    const I8Row r = i8_row(max(max(red[0], red[1]), max(red[2], red[3])));
    for (int k = tid; k < Kp; k += 256)
        q[(size_t)blockIdx.x * ldq + k] = (int8_t)(k < K ? i8_codes(i8_load(x, base + k, type), 0.f, 0.f, 0.f, r) & 0xFFu : 0u);
    if (tid == 0) scale[blockIdx.x] = r.scale;
}

template <int TPR, int C>
static void launch_quantize_reg(const void* x, int64_t ldx, int type, int8_t* q, int64_t ldq, float* scale, int rows, int K, int Kp, hipStream_t s) {
    const dim3 grid((rows + 256 / TPR - 1) / (256 / TPR));
    if (type == FBHIP_F32) hipLaunchKernelGGL((quantize_rows_reg_kernel<TPR, C, true>), grid, dim3(256), 0, s, x, ldx, type, q, ldq, scale, rows, K, Kp);
    else hipLaunchKernelGGL((quantize_rows_reg_kernel<TPR, C, false>), grid, dim3(256), 0, s, x, ldx, type, q, ldq, scale, rows, K, Kp);
}

static void launch_quantize_some(const void* x, int64_t ldx, int type, int8_t* q, int64_t ldq, float* scale, int rows, int K, int Kp, hipStream_t s) {
    const int V = type == FBHIP_F32 ? 4 : 8, pieces = (Kp + V - 1) / V;
    const bool even = ((uintptr_t)q & 7) == 0 && ldq % 8 == 0 && Kp % 8 == 0;          // the codes' rows take whole pieces
    // a wave for a row while a row fits, unless the rows are so few that more threads a row fill the CUs sooner
    if (even && pieces <= 64 * 2) launch_quantize_reg<64, 2>(x, ldx, type, q, ldq, scale, rows, K, Kp, s);
    else if (even && pieces <= 64 * 4 && rows >= 2048) launch_quantize_reg<64, 4>(x, ldx, type, q, ldq, scale, rows, K, Kp, s);
    else if (even && pieces <= 256) launch_quantize_reg<256, 1>(x, ldx, type, q, ldq, scale, rows, K, Kp, s);
    else if (even && pieces <= 256 * 4) launch_quantize_reg<256, 4>(x, ldx, type, q, ldq, scale, rows, K, Kp, s);
    else if (even && pieces <= 256 * 8) launch_quantize_reg<256, 8>(x, ldx, type, q, ldq, scale, rows, K, Kp, s);
    else hipLaunchKernelGGL(quantize_rows_kernel, dim3(rows), dim3(256), 0, s, x, ldx, type, q, ldq, scale, K, Kp);
}

hipError_t launch_quantize_rows(const void* x, int64_t ldx, int type, int8_t* q, int64_t ldq, float* scale, int rows, int K, int Kp, hipStream_t s) {
    constexpr int MOST = 1 << 23;                         // rows of a launch, which may have 2^32 - 1 threads
    for (int64_t r = 0; r < rows; r += MOST)
        launch_quantize_some((const char*)x + r * ldx * (type == FBHIP_F32 ? 4 : 2), ldx, type, q + r * ldq, ldq, scale + r, (int)std::min<int64_t>(MOST, rows - r),
                             K, Kp, s);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------------------------ epilogue
// A scale whose product with any other such scale is a normal number.
__device__ __forceinline__ bool i8_ordinary(float s) { return fabsf(s) >= 0x1p-62f && fabsf(s) <= 0x1p62f; }

// Four neighbouring channels of a token.  The scales' product comes first: neither scale times the sum need be in range.  Where that product itself is no
// normal number (a sum of 0 would make NaN of an infinite one, and a subnormal one has lost bits that a sum of up to 2^31 brings back) the scales'
// exponents are kept apart and applied at the end.
template <bool ORDINARY>
__device__ __forceinline__ void i8_values(const I8Problem& p, const intx4& acc, float sa, const float (&sw)[4], const float (&bias)[4], float (&y)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float s = sa * sw[j];
        y[j] = fmaf((float)acc[j], s, bias[j]);          // (written out: a value must not depend on which of the two forms its tile takes)
        if (!ORDINARY && !__builtin_amdgcn_classf(s, 0x108))          // (a normal number of either sign)
            y[j] = __builtin_amdgcn_ldexpf((float)acc[j] * (__builtin_amdgcn_frexp_mantf(sa) * __builtin_amdgcn_frexp_mantf(sw[j])),
                                           __builtin_amdgcn_frexp_expf(sa) + __builtin_amdgcn_frexp_expf(sw[j])) + bias[j];
        y[j] = p.relu && y[j] < 0.f ? 0.f : y[j];          // (NaN stays)
    }
}

__device__ __forceinline__ uint32_t i8_half(float y, int type) {
    if (type == FBHIP_BF16) {
        const uint32_t b = __float_as_uint(y);
        return y != y ? 0x7FC0u : (b + 0x7FFFu + ((b >> 16) & 1u)) >> 16;       // nearest, ties to even
    }
    const _Float16 f = (_Float16)y;
    uint16_t u;
    __builtin_memcpy(&u, &f, 2);
    return u;
}

__device__ __forceinline__ float i8_channel(const float* v, int n, int N) { return v != nullptr ? v[min(n, N - 1)] : 0.f; }

// Up to four neighbouring values of a row, in one store whatever the row's alignment.
__device__ __forceinline__ void i8_store4(const I8Problem& p, size_t at, int count, const float (&y)[4]) {
    if (p.ytype == FBHIP_F32) {
        float* o = (float*)p.y + at;
        if (count == 4) *(floatx4_any*)o = floatx4_any{y[0], y[1], y[2], y[3]};
        else {
            o[0] = y[0];
            if (count > 1) o[1] = y[1];
            if (count > 2) o[2] = y[2];
        }
        return;
    }
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = i8_half(y[j], p.ytype);
    uint16_t* o = (uint16_t*)p.y + at;
    if (count == 4) *(uintx2_any*)o = uintx2_any{h[0] | h[1] << 16, h[2] | h[3] << 16};
    else {
        o[0] = (uint16_t)h[0];
        if (count > 1) o[1] = (uint16_t)h[1];
        if (count > 2) o[2] = (uint16_t)h[2];
    }
}

template <int COLS, bool ORDINARY>
__device__ __forceinline__ void i8_rows_out(const I8Problem& p, const int* box, int ld, int m, int n, int rows, int cols, const float* sa, const float* sw,
                                            const float* bias, int lane) {
    constexpr int LANES = COLS / 4;
    const int c = lane % LANES * 4;
    if (c >= cols) return;
    const float4 s4 = *(const float4*)(sw + c), b4 = *(const float4*)(bias + c);
    const float s[4] = {s4.x, s4.y, s4.z, s4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll 4
    for (int r = lane / LANES; r < rows; r += 64 / LANES) {
        const intx4 v = *(const intx4*)(box + r * ld + c);
        float y[4];
        i8_values<ORDINARY>(p, v, sa[r], s, b, y);
        i8_store4(p, (size_t)(m + r) * p.ldy + n + c, min(4, cols - c), y);
    }
}

// `rows` tokens from m on, `cols` channels from n on (at most 32 x COLS), their sums in shared memory; the scales and the bias in shared memory too
template <int COLS>
__device__ __forceinline__ void i8_rows(const I8Problem& p, const int* box, int ld, int m, int n, int rows, int cols, const float* sa, const float* sw,
                                        const float* bias, int lane) {
    if (p.partial != nullptr) {          // a slice of K: the sums themselves, rows padded to four
        const int ldp = (p.N + 3) & ~3;
        constexpr int LANES = COLS / 4;
        int* o = p.partial + ((size_t)blockIdx.y * p.M + m) * ldp + n;
        const int c = lane % LANES * 4;
        if (c < cols)
#pragma unroll 4
            for (int r = lane / LANES; r < rows; r += 64 / LANES) *(intx4*)(o + (size_t)r * ldp + c) = *(const intx4*)(box + r * ld + c);
        return;
    }
    // (asked once for all: a test of each product in the loop costs 3 % of 2500 x 5001 x 1999)
    bool ordinary = i8_ordinary(sa[lane & 31]);
#pragma unroll
    for (int c = 0; c < COLS; c += 64) ordinary = ordinary && i8_ordinary(sw[c + (COLS < 64 ? lane & (COLS - 1) : lane)]);
    if (__all(ordinary)) i8_rows_out<COLS, true>(p, box, ld, m, n, rows, cols, sa, sw, bias, lane);
    else i8_rows_out<COLS, false>(p, box, ld, m, n, rows, cols, sa, sw, bias, lane);
}

// the last `valid` (1..15, or more: all) of a lane's 16 codes of the K dimension stay
__device__ __forceinline__ intx4 i8_mask(intx4 v, int valid) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int left = valid - 4 * j;
        v[j] = left >= 4 ? v[j] : left <= 0 ? 0 : v[j] & (int)((1u << (8 * left)) - 1u);
    }
    return v;
}

// ------------------------------------------------------------------------------------------------------------------ tiles
// A workgroup of WN x WM waves computes a tile of (WN FN 32) channels x (WM FM 32) tokens; a wave keeps FN x FM accumulators of the
// 32x32x32 matrix instruction, the weights as its first operand, so that a lane holds four neighbouring channels of one token.
// Measured from codes, back to back on one input (us, fp32 out): 8192^3 480 (2.29 PTOPS; the clock falls to 1.7 GHz, matrix instructions alone on such
// operands reach 3.45), 4096^3 67-70 (1.66 a step of 128 and 15 for start and output), 2500 x 5001 x 1999 37-40, 4096 x 2048 x 2048 24-26,
// 1024 x 2048 x 1024 8.3.  Inputs in turn and launches apart cost more: 8192^3 with three inputs 500-505, one launch after a pause 532, under a trace 538-566.
// A step takes BK bytes of K: both operands' rows of it come straight into shared memory (16 bytes a lane), S steps deep.  Shared memory
// has 64 banks: a fragment read of 16 rows' 16-byte pieces is free of conflicts if rows that lie a multiple of 256 bytes apart keep them in
// different places, so the pieces of row r are stored in the order piece ^ (r / (256 / BK)).
template <int WN, int WM, int FN, int FM, int BK_, int S_>
struct I8Tile {
    static constexpr int WAVES = WN * WM, THREADS = 64 * WAVES, BN = WN * FN * 32, BM = WM * FM * 32, ROWS = BN + BM, BK = BK_, S = S_;
    static constexpr int PER_ROW = BK / 16, PIECE_ROWS = 64 / PER_ROW;      // 16-byte pieces of a row; rows of a 1 KB load
    static constexpr int PIECES = ROWS / PIECE_ROWS / WAVES;                // loads a wave issues for a step
    static constexpr int SLICES = BK / 32, STAGE = ROWS * BK;
    static constexpr int BOX_LD = FN * 32 + 4, BOX = 32 * BOX_LD * 4;       // a wave's 32 tokens on their way out
    static constexpr int TILES = S * STAGE > WAVES * BOX ? S * STAGE : WAVES * BOX, LDS = TILES + (2 * BN + BM) * 4;
    static_assert(ROWS % (PIECE_ROWS * WAVES) == 0 && LDS <= 160 * 1024 && (BK == 64 || BK == 128), "tile");
    static __device__ __forceinline__ int place(int row, int piece) { return (piece ^ ((row / (256 / BK)) & (PER_ROW - 1))) * 16; }
};

// 1 KB of global memory into shared memory, lane l's 16 bytes behind lane l-1's.  (Assembly: the compiler would wait for all such
// loads in front of every read of shared memory; no register is written.)
__device__ __forceinline__ void i8_load_lds(uint32_t lds, uint32_t offset, const void* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}

template <int COUNT>
__device__ __forceinline__ void i8_wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(COUNT) : "memory"); }

// The operands of one matrix instruction along K (32 codes), slice kk of a step: `w0` / `a0` is where the lane's first row keeps its piece of
// slice 0; the rows of the other fragments lie 32 rows on, and slice kk's piece is 2 kk pieces away, by exclusive or.
template <class T, int FN, int FM>
__device__ __forceinline__ void i8_fragments(const int8_t* st, int kk, uint32_t w0, uint32_t a0, intx4 (&w)[FN], intx4 (&a)[FM]) {
    const int8_t *wp = st + (w0 ^ (kk * 32)), *ap = st + (a0 ^ (kk * 32));
#pragma unroll
    for (int i = 0; i < FN; ++i) w[i] = *(const intx4*)(wp + i * 32 * T::BK);
#pragma unroll
    for (int j = 0; j < FM; ++j) a[j] = *(const intx4*)(ap + j * 32 * T::BK);
}

template <int WN, int WM, int FN, int FM, int BK, int S>
__global__ void __launch_bounds__((I8Tile<WN, WM, FN, FM, BK, S>::THREADS), (FN * FM <= 4 ? 4 : 2)) gemm_i8_kernel(const I8Problem p) {
    using T = I8Tile<WN, WM, FN, FM, BK, S>;
    extern __shared__ __attribute__((aligned(1024))) int8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_n = (p.N + T::BN - 1) / T::BN, tiles_m = (p.M + T::BM - 1) / T::BM, tiles = tiles_n * tiles_m;
    // workgroup b runs on XCD b % 8: each XCD takes one run of the tiles
    const int xcd = blockIdx.x & 7, each = tiles >> 3, rest = tiles & 7;
    const int t = (xcd < rest ? xcd * (each + 1) : rest * (each + 1) + (xcd - rest) * each) + ((int)blockIdx.x >> 3);
    // ... in blocks of a few token tiles, so that its 32 CUs share 4 + 8 (or 8 + 4) tiles' operands and not 1 + 32.  8192^3: 479 us with four
    // token tiles of 256, 484 with eight; 4096 x 2048 x 2048: 24.1 with eight of 128, 24.5 with four
    constexpr int GROUP = T::BM == 256 ? 4 : 8;
    const int group = t / (GROUP * tiles_n), g0 = group * GROUP, gm = min(GROUP, tiles_m - g0), in_group = t - group * GROUP * tiles_n;
    const int n0 = (in_group / gm) * T::BN, m0 = (g0 + in_group % gm) * T::BM;
    const int steps_all = (p.K + BK - 1) / BK;
    const int k_first = blockIdx.y * p.steps, steps = min(p.steps, steps_all - k_first);
    const bool tail = k_first + steps == steps_all && (p.K & (BK - 1)) != 0;

    // where this lane loads from: row lane / PER_ROW of each 1 KB of rows
    uint32_t off[T::PIECES];
#pragma unroll
    for (int q = 0; q < T::PIECES; ++q) {
        const int row = (wave * T::PIECES + q) * T::PIECE_ROWS + lane / T::PER_ROW, c16 = T::place(row, lane % T::PER_ROW);
        off[q] = row < T::BN ? (uint32_t)min(row, p.N - 1 - n0) * (uint32_t)p.ldw + c16 : (uint32_t)min(row - T::BN, p.M - 1 - m0) * (uint32_t)p.lda + c16;
    }
    const int8_t* wbase = p.w + (size_t)n0 * p.ldw;
    const int8_t* abase = p.a + (size_t)m0 * p.lda;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) int8_t*)smem;
    // the last step of an uneven K reads no further than the 16 bytes that hold the row's end
    const int k16 = (p.K + 15) & ~15, last_piece = k16 - 16 - (steps_all - 1) * BK;
    auto issue = [&](int s, int q) __attribute__((always_inline)) {
        const int piece = wave * T::PIECES + q;
        uint32_t from = off[q];
        if (tail && s == steps - 1) {
            const int row = piece * T::PIECE_ROWS + lane / T::PER_ROW;
            from -= (uint32_t)max(0, T::place(row, lane % T::PER_ROW) - last_piece);
        }
        i8_load_lds(lds0 + (uint32_t)((s % S) * T::STAGE + piece * 1024), from, (piece * T::PIECE_ROWS < T::BN ? wbase : abase) + (size_t)(k_first + s) * BK);
    };

    // the tile's scales and bias: their loads go first; at the end they lie behind the tiles, where a lane finds its 4 FN channels' and FM tokens'
    float *sw = (float*)(smem + T::TILES), *bias = sw + T::BN, *sa = bias + T::BN;
    static_assert(T::THREADS >= T::BN && T::THREADS >= T::BM, "a thread for each channel and token of the tile");
    const float edge_sw = i8_channel(p.sw, n0 + (int)threadIdx.x, p.N), edge_bias = i8_channel(p.bias, n0 + (int)threadIdx.x, p.N);
    const float edge_sa = i8_channel(p.sa, m0 + (int)threadIdx.x, p.M);

    const int l31 = lane & 31, half = lane >> 5, wn = wave % WN, wm = wave / WN;
    const int wrow = wn * FN * 32 + l31, arow = T::BN + wm * FM * 32 + l31;
    const uint32_t w0 = wrow * BK + T::place(wrow, half), a0 = arow * BK + T::place(arow, half);
    intx16 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

    // The fragments of a slice are read while the slice before it is multiplied.  Before the last slice of a step everybody has read the
    // step's tile, and the next step's has landed: step s + S goes into the place of step s, its loads spread over a step's slices.
    const int full = steps - (tail ? 1 : 0);
    intx4 w[2][FN], a[2][FM];
#pragma unroll
    for (int s = 0; s < S; ++s)
        if (s < steps) {
#pragma unroll
            for (int q = 0; q < T::PIECES; ++q) issue(s, q);
        }
    if (steps >= S) i8_wait_loads<(S - 1) * T::PIECES>();
    else i8_wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    i8_fragments<T>(smem, 0, w0, a0, w[0], a[0]);
    // slice `set`'s products, with share r of the loads of step `to` between them
    auto multiply = [&](int set, int r, int to) __attribute__((always_inline)) {
        const bool live = to >= S && to < steps;
        const int first = r * T::PIECES / T::SLICES, count = (r + 1) * T::PIECES / T::SLICES - first;
        int done = 0;
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[set][i], a[set][j], acc[i][j], 0, 0, 0);
                if (done * FN * FM < (i * FM + j + 1) * count) {
                    if (live) issue(to, first + done);
                    ++done;
                }
            }
    };
    for (int s = 0; s < full; ++s) {
        const int8_t *st = smem + (s % S) * T::STAGE, *next = smem + ((s + 1) % S) * T::STAGE;
#pragma unroll
        for (int kk = 0; kk + 1 < T::SLICES; ++kk) {
            i8_fragments<T>(st, kk + 1, w0, a0, w[(kk + 1) & 1], a[(kk + 1) & 1]);
            multiply(kk & 1, kk + 1, s - 1 + S);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (s + S <= steps) i8_wait_loads<(S - 2) * T::PIECES>();
        else i8_wait_loads<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        i8_fragments<T>(next, 0, w0, a0, w[0], a[0]);       // (behind the last step: not used)
        multiply((T::SLICES - 1) & 1, 0, s + S);
    }
    if (tail) {          // only `left` codes of the last step belong to K; the other operand may hold anything behind them
        const int left = p.K - (steps_all - 1) * BK;
#pragma unroll
        for (int kk = 0; kk < T::SLICES; ++kk) {
            i8_fragments<T>(smem + (full % S) * T::STAGE, kk, w0, a0, w[0], a[0]);
#pragma unroll
            for (int j = 0; j < FM; ++j) a[0][j] = i8_mask(a[0][j], left - (2 * kk + half) * 16);
            multiply(0, 0, 0);
        }
    }
    // A wave's 32 tokens at a time go through its own part of shared memory, so that its stores are whole lines of a token's row, whatever the
    // row's alignment: a lane's accumulators lie 32 tokens apart.
    if ((int)threadIdx.x < T::BN) { sw[threadIdx.x] = edge_sw; bias[threadIdx.x] = edge_bias; }
    if ((int)threadIdx.x < T::BM) sa[threadIdx.x] = edge_sa;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    int* box = (int*)(smem + wave * T::BOX);
    const int nw = wn * FN * 32;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const intx4 c = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                *(intx4*)(box + l31 * T::BOX_LD + i * 32 + 8 * g + 4 * half) = c;
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const int mt = (wm * FM + j) * 32;
        const int rows = min(32, p.M - m0 - mt), cols = min(FN * 32, p.N - n0 - nw);
        if (rows > 0 && cols > 0) i8_rows<FN * 32>(p, box, T::BOX_LD, m0 + mt, n0 + nw, rows, cols, sa + mt, sw + nw, bias + nw, lane);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// the sums of a K that was split over several workgroups
__global__ void __launch_bounds__(256) gemm_i8_fold_kernel(const I8Problem p, int slices) {
    const int quads = (p.N + 3) / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)p.M * quads) return;
    const int m = (int)(i / quads), n = (int)(i % quads) * 4;
    intx4 acc = {0, 0, 0, 0};
    for (int s = 0; s < slices; ++s) acc += *(const intx4*)(p.partial + ((size_t)s * p.M + m) * (quads * 4) + n);
    float y[4], sw[4], bias[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) { sw[j] = i8_channel(p.sw, n + j, p.N); bias[j] = i8_channel(p.bias, n + j, p.N); }
    i8_values<false>(p, acc, p.sa[m], sw, bias, y);
    i8_store4(p, (size_t)m * p.ldy + n, min(4, p.N - n), y);
}

// ------------------------------------------------------------------------------------------------------------------ few tokens
// Few tokens: what counts is the weights' way from memory.  A workgroup of eight waves takes 16 NT channels and up to 16 MT tokens, its waves 128
// codes of K in turn, both operands straight from memory into the 16x16x64 matrix instruction (a lane's 32 codes in a row are two
// instructions' share: the operands agree on the order of K, which is all that the sum asks for).  The eight partial sums are added in shared memory.
// Measured from codes, back to back (us): 5 tokens 1024 x 1024 2.8, 4096 x 4096 5.2, 8192 x 8192 14.0 (67 MB of weights, 4.8 TB/s).
// TOKENS > 0: up to that many tokens are quantised by every workgroup for itself, while its first weights are on their way: a launch less.
constexpr int I8_STRIP_MOST = 1 << 26;                    // channels of a launch of strips, which may have 2^32 - 1 threads (tiles take more)
constexpr int I8_STRIP_WAVES = 8, I8_STRIP_THREADS = 64 * I8_STRIP_WAVES, I8_STRIP_VALUES = 32;      // values of x that a thread holds

// TOKENS rows of x into codes [TOKENS][Kp] and scales in shared memory; 512 / TOKENS threads a row, I8_STRIP_VALUES values a thread
template <int TOKENS, bool WIDE>
__device__ __forceinline__ void i8_strip_quantize(const I8Problem& p, const void* x, int64_t ldx, int type, int8_t* codes, int Kp, float* scale,
                                                  uint32_t* red) {
    constexpr int V = WIDE ? 4 : 8, C = I8_STRIP_VALUES / V, TPT = I8_STRIP_THREADS / TOKENS, WPT = TPT / 64;
    const int tid = threadIdx.x, m = tid / TPT, t = tid % TPT;
    const char* base = (const char*)x + (size_t)min(m, p.M - 1) * ldx * (16 / V);
    uint4 raw[C];
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) raw[c] = i8_piece<WIDE>(base, (c * TPT + t) * V, p.K);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
        for (int e = 0; e < V; ++e) top = i8_top(top, i8_unpack<WIDE>(w, e, type));
    }
    top = i8_lanes_top<TPT < 64 ? TPT : 64>(top);
    if (WPT > 1) {                        // several waves hold the token
        if ((tid & 63) == 0) red[tid >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int q = 0; q < WPT; ++q) top = max(top, red[m * WPT + q]);
    }
    const I8Row r = i8_row(top);
    if (t == 0) scale[m] = r.scale;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int k = (c * TPT + t) * V;
        if (k >= Kp) break;
        const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
        for (int e = 0; e < V; e += 4)
            *(uint32_t*)(codes + m * Kp + k + e) = i8_codes(i8_unpack<WIDE>(w, e, type), i8_unpack<WIDE>(w, e + 1, type), i8_unpack<WIDE>(w, e + 2, type),
                                                            i8_unpack<WIDE>(w, e + 3, type), r);
    }
    __syncthreads();
}

template <int NT, int MT, int TOKENS>
__global__ void __launch_bounds__(I8_STRIP_THREADS) gemm_i8_strip_kernel(const I8Problem p, const void* __restrict__ x, int64_t ldx, int xtype) {
    static_assert(TOKENS <= 16 && (TOKENS == 0 || MT == 1), "quantised tokens fit one tile");
    extern __shared__ __attribute__((aligned(16))) int8_t codes[];         // TOKENS > 0: [TOKENS][Kp]
    __shared__ __attribute__((aligned(16))) intx4 part[I8_STRIP_WAVES][NT * MT][64];
    __shared__ float token_scale[16];
    __shared__ uint32_t red[I8_STRIP_WAVES];
    constexpr int DEEP = NT * MT >= 4 ? 2 : 4;                // chunks whose loads are under way together
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, quarter = lane >> 4;
    const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT, K = p.K, chunks = (K + 127) / 128, k16 = (K + 15) & ~15, Kp = chunks * 128;
    const int8_t *wp[NT], *ap[MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) wp[i] = p.w + (size_t)min(n0 + 16 * i + l15, p.N - 1) * p.ldw;
#pragma unroll
    for (int j = 0; j < MT; ++j) ap[j] = TOKENS ? codes + l15 * Kp : p.a + (size_t)min(m0 + 16 * j + l15, p.M - 1) * p.lda;
    intx4 acc[NT][MT], w[DEEP][NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = intx4{0, 0, 0, 0};
    auto load = [&](int c0) __attribute__((always_inline)) {
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            if (c0 + d * I8_STRIP_WAVES >= chunks) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = min((c0 + d * I8_STRIP_WAVES) * 128 + quarter * 32 + h * 16, k16 - 16);
#pragma unroll
                for (int i = 0; i < NT; ++i) w[d][i][h] = *(const intx4*)(wp[i] + k);
            }
        }
    };
    load(wave);
    if (TOKENS) {
        if (xtype == FBHIP_F32) i8_strip_quantize<TOKENS ? TOKENS : 1, true>(p, x, ldx, xtype, codes, Kp, token_scale, red);
        else i8_strip_quantize<TOKENS ? TOKENS : 1, false>(p, x, ldx, xtype, codes, Kp, token_scale, red);
    }
    for (int c0 = wave; c0 < chunks; c0 += I8_STRIP_WAVES * DEEP) {
        intx4 a[DEEP][MT][2];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const int c = c0 + d * I8_STRIP_WAVES;
            if (c >= chunks) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = c * 128 + quarter * 32 + h * 16;
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    if (TOKENS) a[d][j][h] = l15 < TOKENS ? *(const intx4*)(ap[j] + k) : intx4{0, 0, 0, 0};
                    else a[d][j][h] = *(const intx4*)(ap[j] + min(k, k16 - 16));
                }
            }
        }
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const int c = c0 + d * I8_STRIP_WAVES;
            if (c >= chunks) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (!TOKENS && c == chunks - 1 && (K & 127)) {          // codes behind K count nothing, whatever the weights hold there
#pragma unroll
                    for (int j = 0; j < MT; ++j) a[d][j][h] = i8_mask(a[d][j][h], K - (c * 128 + quarter * 32 + h * 16));
                }
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int j = 0; j < MT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[d][i][h], a[d][j][h], acc[i][j], 0, 0, 0);
            }
        }
        if (c0 + I8_STRIP_WAVES * DEEP < chunks) load(c0 + I8_STRIP_WAVES * DEEP);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) part[wave][i * MT + j][lane] = acc[i][j];
    __syncthreads();
    for (int q = threadIdx.x; q < NT * MT * 64; q += I8_STRIP_THREADS) {
        const int f = q >> 6, l = q & 63, m = m0 + 16 * (f % MT) + (l & 15), n = n0 + 16 * (f / MT) + 4 * (l >> 4);
        if (m >= p.M || n >= p.N) continue;
        intx4 v = part[0][f][l];
#pragma unroll
        for (int u = 1; u < I8_STRIP_WAVES; ++u) v += part[u][f][l];
        float y[4], sw[4], bias[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) { sw[e] = i8_channel(p.sw, n + e, p.N); bias[e] = i8_channel(p.bias, n + e, p.N); }
        i8_values<false>(p, v, TOKENS ? token_scale[m] : p.sa[m], sw, bias, y);
        i8_store4(p, (size_t)m * p.ldy + n, min(4, p.N - n), y);
    }
}

// ------------------------------------------------------------------------------------------------------------------ choice
template <int WN, int WM, int FN, int FM, int BK, int S>
static hipError_t launch_i8_tile(I8Problem p, int slices, hipStream_t s) {
    using T = I8Tile<WN, WM, FN, FM, BK, S>;
    // the limit of dynamic shared memory belongs to the current device's copy of the kernel: it is raised once on each (twice does no harm)
    static std::atomic<uint64_t> ready{0};
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    if (dev < 0 || dev >= 64) return hipErrorInvalidDevice;
    if (!(ready.load(std::memory_order_relaxed) >> dev & 1)) {
        e = hipFuncSetAttribute(reinterpret_cast<const void*>(&gemm_i8_kernel<WN, WM, FN, FM, BK, S>), hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS);
        if (e != hipSuccess) return e;
        ready.fetch_or((uint64_t)1 << dev, std::memory_order_relaxed);
    }
    const int tiles = ((p.N + T::BN - 1) / T::BN) * ((p.M + T::BM - 1) / T::BM);
    p.steps *= I8_BK / BK;
    hipLaunchKernelGGL((gemm_i8_kernel<WN, WM, FN, FM, BK, S>), dim3(tiles, slices), dim3(T::THREADS), T::LDS, s, p);
    return hipGetLastError();
}

// Which kernel.  Measured with fp32 outputs, from codes, launches back to back in a graph (us):
//   strips up to 16 tokens, and up to 64 where the weights take up to 32 MB: 1024 x 1024 with 64 tokens 4.6 (tile 6.3), 4096 x 4096 with 64 tokens
//   11.9 (tile 13), 8192 x 8192 with 32 tokens 21.4 (tile 16.6); a long K with few channels is for the tiles, which can split it: 64 x 64 x 65536 140 as
//   four strips;
//   256 x 256 from 192 tiles on: 2500 x 5001 x 1999 (200 tiles) 42.8, 128 x 128 47.8; with 128 tiles (4096 x 2048 x 2048) 32.0 and 24.5;
//   128 x 128 from 192 tiles on: 2048 x 2048 x 1024 (256 tiles) 11.1, 64 x 64 12.5; with 128 tiles (1024 x 2048 x 1024) 9.4 and 8.2;
//   64 x 64 below, four steps deep while two such workgroups a CU are enough: 256 x 4096 x 4096 13.1, two steps deep 14.9; 1024 tiles
//   (2048 x 2048 x 1024) 14.1 and 12.5.  K over several workgroups costs 4 us for the second launch and saves 0.28 us a step: from 32 steps
//   and with CUs to spare only.
I8Plan gemm_i8_plan(int M, int N, int K) {
    I8Plan plan{};
    const int steps = (K + I8_BK - 1) / I8_BK;
    plan.slices = 1;
    plan.steps = steps;
    const bool long_k = K > 16384 && N < 2048;
    if (!long_k && N <= I8_STRIP_MOST && (M <= 16 || (M <= 64 && (int64_t)N * K <= (int64_t)1 << 25))) { plan.tile = 16; return plan; }
    const int64_t t256 = (int64_t)((M + 255) / 256) * ((N + 255) / 256), t128 = (int64_t)((M + 127) / 128) * ((N + 127) / 128);
    const int64_t t64 = (int64_t)((M + 63) / 64) * ((N + 63) / 64);
    if (t256 >= 192) plan.tile = 256;
    else if (t128 >= 192) plan.tile = 128;
    else {
        plan.tile = 64;
        if (t64 <= 128 && steps >= 32) plan.slices = (int)std::min<int64_t>(256 / t64, steps / 8);
        plan.steps = (steps + plan.slices - 1) / plan.slices;
        plan.slices = (steps + plan.steps - 1) / plan.steps;
        plan.deep = t64 * plan.slices <= 512;
    }
    return plan;
}

template <int NT, int MT>
static void launch_i8_strip(const I8Problem& p, hipStream_t s) {
    hipLaunchKernelGGL((gemm_i8_strip_kernel<NT, MT, 0>), dim3((p.N + 16 * NT - 1) / (16 * NT), (p.M + 16 * MT - 1) / (16 * MT)), dim3(I8_STRIP_THREADS), 0, s, p,
                       nullptr, (int64_t)0, (int)FBHIP_F32);
}

// Up to 16 tokens (as 1, 2, 4, 8 or 16) whose values fit I8_STRIP_VALUES a thread are quantised by every workgroup of the product.  With 128 values a
// thread more of them fit, but 4 tokens of 8192 values took 29 us in one launch and 18 in two.
static int i8_tokens(int M) { return M <= 2 ? M : M <= 4 ? 4 : M <= 8 ? 8 : 16; }

bool linear_i8_fused(int M, int N, int K) { return M <= 16 && N <= I8_STRIP_MOST && K <= I8_STRIP_VALUES * I8_STRIP_THREADS / i8_tokens(M); }

template <int TOKENS>
static hipError_t launch_i8_strip_tokens(const I8Problem& p, const void* x, int64_t ldx, int xtype, hipStream_t s) {
    const size_t lds = (size_t)TOKENS * ((p.K + 127) / 128 * 128);         // at most I8_STRIP_VALUES * I8_STRIP_THREADS bytes
    hipLaunchKernelGGL((gemm_i8_strip_kernel<1, 1, TOKENS>), dim3((p.N + 15) / 16), dim3(I8_STRIP_THREADS), lds, s, p, x, ldx, xtype);
    return hipGetLastError();
}

hipError_t launch_linear_i8_tokens(I8Problem p, const void* x, int64_t ldx, int xtype, hipStream_t s) {
    switch (i8_tokens(p.M)) {
        case 1: return launch_i8_strip_tokens<1>(p, x, ldx, xtype, s);
        case 2: return launch_i8_strip_tokens<2>(p, x, ldx, xtype, s);
        case 4: return launch_i8_strip_tokens<4>(p, x, ldx, xtype, s);
        case 8: return launch_i8_strip_tokens<8>(p, x, ldx, xtype, s);
        default: return launch_i8_strip_tokens<16>(p, x, ldx, xtype, s);
    }
}

hipError_t launch_gemm_i8(I8Problem p, int* partial, hipStream_t s) {
    const I8Plan plan = gemm_i8_plan(p.M, p.N, p.K);
    if (plan.tile == 16) {
        const bool wide = p.N >= 8192;
        if (p.M <= 16) launch_i8_strip<1, 1>(p, s);
        else if (p.M <= 32) wide ? launch_i8_strip<2, 2>(p, s) : launch_i8_strip<1, 2>(p, s);
        else wide ? launch_i8_strip<2, 4>(p, s) : launch_i8_strip<1, 4>(p, s);
        return hipGetLastError();
    }
    p.steps = plan.steps;
    p.partial = plan.slices > 1 ? partial : nullptr;
    hipError_t e;
    if (plan.tile == 256) e = launch_i8_tile<2, 4, 4, 2, 128, 2>(p, plan.slices, s);
    else if (plan.tile == 128) e = launch_i8_tile<2, 4, 2, 1, 128, 2>(p, plan.slices, s);
    else if (plan.deep) e = launch_i8_tile<2, 2, 1, 1, 128, 4>(p, plan.slices, s);
    else e = launch_i8_tile<2, 2, 1, 1, 128, 2>(p, plan.slices, s);
    if (e != hipSuccess || plan.slices == 1) return e;
    const int64_t quads = (int64_t)p.M * ((p.N + 3) / 4);
    hipLaunchKernelGGL(gemm_i8_fold_kernel, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, p, plan.slices);
    return hipGetLastError();
}

}  // namespace fbhip
