// Matrix product in 8-bit integers: y[m, n] = act( (sum_k a[m, k] w[n, k]) * sa[m] * sw[n] + bias[n] ), with a scale for each row of both
// operands, and the row quantiser that makes them: s = max|x| / 127, code = nearest whole number to x / s (ties to even).
//
// The sum is exact: |sum| <= K 127^2 < 2^31 up to K = 131072, the largest that the entry points take, whatever the order of the additions, so K may
// be split at will.  It is turned into a float once (24 bits) and scaled in single precision.
#include "common.h"
#include "host.h"

namespace fbhip {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));

constexpr int I8_BK = 128;                    // bytes of K in a step: one row of a tile is one 128-byte line

// ------------------------------------------------------------------------------------------------------------------ quantiser
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}

__device__ __forceinline__ float i8_load(const void* x, size_t i, int type) {
    if (type == FBHIP_F32) return ((const float*)x)[i];
    const uint16_t h = ((const uint16_t*)x)[i];
    if (type == FBHIP_BF16) return __uint_as_float((uint32_t)h << 16);
    _Float16 f;
    __builtin_memcpy(&f, &h, 2);
    return (float)f;
}

// One workgroup takes a row.  A row that holds a NaN or an infinity gets the scale NaN (and codes 0): its whole output row is NaN.  A row of zeros,
// or one so small that its scale is 0, gets codes 0.
__global__ void __launch_bounds__(256) quantize_rows_kernel(const void* __restrict__ x, int64_t ldx, int type, int8_t* __restrict__ q, int64_t ldq,
                                                            float* __restrict__ scale, int K, int Kp) {
    __shared__ float red[4];
    __shared__ int bad;
    const int tid = threadIdx.x;
    const size_t base = (size_t)blockIdx.x * ldx;
    if (tid == 0) bad = 0;
    __syncthreads();
    float top = 0.f;
    bool odd = false;
    for (int k = tid; k < K; k += 256) {
        const float v = fabsf(i8_load(x, base + k, type));
        odd = odd || !(v < __uint_as_float(0x7F800000u));
        top = fmaxf(top, v);
    }
    top = wave_max(top);
    if ((tid & 63) == 0) red[tid >> 6] = top;
    if (odd) bad = 1;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float s = top / 127.f;
    const bool zero = bad || s == 0.f;
    for (int k = tid; k < Kp; k += 256) {
        float c = 0.f;
        if (k < K && !zero) c = fminf(fmaxf(rintf(i8_load(x, base + k, type) / s), -127.f), 127.f);
        q[(size_t)blockIdx.x * ldq + k] = (int8_t)(int)c;
    }
    if (tid == 0) scale[blockIdx.x] = bad ? __uint_as_float(0x7FC00000u) : s;
}

hipError_t launch_quantize_rows(const void* x, int64_t ldx, int type, int8_t* q, int64_t ldq, float* scale, int rows, int K, int Kp, hipStream_t s) {
    hipLaunchKernelGGL(quantize_rows_kernel, dim3(rows), dim3(256), 0, s, x, ldx, type, q, ldq, scale, K, Kp);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------------------------ epilogue
// y[m, n .. n+3] from the sums of four neighbouring columns
__device__ __forceinline__ void i8_store4(const I8Problem& p, int m, int n, int a0, int a1, int a2, int a3) {
    if (m >= p.M || n >= p.N) return;
    const float sa = p.sa[m];
    const int acc[4] = {a0, a1, a2, a3};
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = min(n + j, p.N - 1);
        y[j] = (float)acc[j] * sa * p.sw[c];
        if (p.bias != nullptr) y[j] += p.bias[c];
        if (p.relu) y[j] = y[j] < 0.f ? 0.f : y[j];          // (NaN stays)
    }
    const size_t at = (size_t)m * p.ldy + n;
    if (p.ytype == FBHIP_F32) {
        float* o = (float*)p.y + at;
        if (p.yvec && n + 3 < p.N) { *(float4*)o = make_float4(y[0], y[1], y[2], y[3]); return; }
        for (int j = 0; j < 4 && n + j < p.N; ++j) o[j] = y[j];
        return;
    }
    uint16_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (p.ytype == FBHIP_BF16) {
            const uint32_t b = __float_as_uint(y[j]);
            h[j] = y[j] != y[j] ? 0x7FC0 : (uint16_t)((b + 0x7FFFu + ((b >> 16) & 1u)) >> 16);       // nearest, ties to even
        } else {
            const _Float16 f = (_Float16)y[j];
            __builtin_memcpy(&h[j], &f, 2);
        }
    }
    uint16_t* o = (uint16_t*)p.y + at;
    if (p.yvec && n + 3 < p.N) { *(uint2*)o = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16); return; }
    for (int j = 0; j < 4 && n + j < p.N; ++j) o[j] = h[j];
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
// Both operands come in rows of 128 bytes straight into shared memory (16 bytes a lane), two steps ahead.  The 16-byte pieces of row r are
// stored in the order piece ^ (r & 7): eight rows' pieces of the same place fall into different banks.
template <int WN, int WM, int FN, int FM>
struct I8Tile {
    static constexpr int WAVES = WN * WM, THREADS = 64 * WAVES, BN = WN * FN * 32, BM = WM * FM * 32, ROWS = BN + BM;
    static constexpr int PIECES = ROWS / 8 / WAVES;            // 1 KB loads a wave issues for a step
    static constexpr int STAGE = ROWS * I8_BK, LDS = 2 * STAGE;
    static_assert(ROWS % (8 * WAVES) == 0 && LDS <= 160 * 1024, "tile");
};

// 1 KB of global memory into shared memory, lane l's 16 bytes behind lane l-1's.  (Assembly: the compiler would wait for all such
// loads in front of every read of shared memory; no register is written.)
__device__ __forceinline__ void i8_load_lds(uint32_t lds, uint32_t offset, const void* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(offset), "s"(base) : "memory");
}

// the operands of one matrix instruction along K (32 codes): slice kk of a step
template <class T, int FN, int FM>
__device__ __forceinline__ void i8_fragments(const int8_t* st, int kk, int wn, int wm, int l31, int half, intx4 (&w)[FN], intx4 (&a)[FM]) {
    const int piece = 2 * kk + half;
#pragma unroll
    for (int i = 0; i < FN; ++i) {
        const int row = (wn * FN + i) * 32 + l31;
        w[i] = *(const intx4*)(st + row * I8_BK + ((piece ^ (row & 7)) * 16));
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const int row = T::BN + (wm * FM + j) * 32 + l31;
        a[j] = *(const intx4*)(st + row * I8_BK + ((piece ^ (row & 7)) * 16));
    }
}

template <int FN, int FM>
__device__ __forceinline__ void i8_multiply(const intx4 (&w)[FN], const intx4 (&a)[FM], intx16 (&acc)[FN][FM]) {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[i], a[j], acc[i][j], 0, 0, 0);
}

// the first step's tile has landed; the second's loads may be under way
template <int PIECES>
__device__ __forceinline__ void i8_wait(bool second) {
    if (second) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PIECES) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <int WN, int WM, int FN, int FM>
__global__ void __launch_bounds__((I8Tile<WN, WM, FN, FM>::THREADS)) gemm_i8_kernel(const I8Problem p) {
    using T = I8Tile<WN, WM, FN, FM>;
    extern __shared__ __attribute__((aligned(1024))) int8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_n = (p.N + T::BN - 1) / T::BN, tiles_m = (p.M + T::BM - 1) / T::BM, tiles = tiles_n * tiles_m;
    // workgroup b runs on XCD b % 8: each XCD takes one run of the tiles
    const int xcd = blockIdx.x & 7, each = tiles >> 3, rest = tiles & 7;
    const int t = (xcd < rest ? xcd * (each + 1) : rest * (each + 1) + (xcd - rest) * each) + ((int)blockIdx.x >> 3);
    // ... in blocks of eight token tiles, so that its 32 CUs share 8 + 4 tiles' operands and not 1 + 32
    const int group = t / (8 * tiles_n), g0 = group * 8, gm = min(8, tiles_m - g0), in_group = t - group * 8 * tiles_n;
    const int n0 = (in_group / gm) * T::BN, m0 = (g0 + in_group % gm) * T::BM;
    const int steps_all = (p.K + I8_BK - 1) / I8_BK;
    const int k_first = blockIdx.y * p.steps, steps = min(p.steps, steps_all - k_first);
    const bool tail = k_first + steps == steps_all && (p.K & (I8_BK - 1)) != 0;

    // where this lane loads from: row (lane >> 3) of each 8-row piece, 16-byte piece (lane & 7) ^ row
    const int r8 = lane >> 3, c16 = ((lane & 7) ^ r8) * 16;
    uint32_t off[T::PIECES];
#pragma unroll
    for (int q = 0; q < T::PIECES; ++q) {
        const int row = (wave * T::PIECES + q) * 8 + r8;
        off[q] = row < T::BN ? (uint32_t)min(row, p.N - 1 - n0) * (uint32_t)p.ldw + c16 : (uint32_t)min(row - T::BN, p.M - 1 - m0) * (uint32_t)p.lda + c16;
    }
    // the last step of an uneven K reads no further than the 16 bytes that hold the row's end
    const int k16 = (p.K + 15) & ~15;
    const uint32_t back = (uint32_t)max(0, (steps_all - 1) * I8_BK + c16 - (k16 - 16));
    const int8_t* wbase = p.w + (size_t)n0 * p.ldw;
    const int8_t* abase = p.a + (size_t)m0 * p.lda;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) int8_t*)smem;
    auto issue = [&](int s) __attribute__((always_inline)) {
        const uint32_t minus = tail && s == steps - 1 ? back : 0u;
        const size_t k = (size_t)(k_first + s) * I8_BK;
#pragma unroll
        for (int q = 0; q < T::PIECES; ++q) {
            const int piece = wave * T::PIECES + q;
            i8_load_lds(lds0 + (uint32_t)((s & 1) * T::STAGE + piece * 1024), off[q] - minus, (piece * 8 < T::BN ? wbase : abase) + k);
        }
    };

    const int l31 = lane & 31, half = lane >> 5, wn = wave % WN, wm = wave / WN;
    intx16 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

    // The fragments of a slice are read while the slice before it is multiplied.  Before the last slice of a step everybody has read the
    // step's tile, and the next step's has landed: the one after it goes into the same place, with a whole step's time to arrive.
    const int full = steps - (tail ? 1 : 0);
    intx4 w[2][FN], a[2][FM];
    issue(0);
    if (steps > 1) issue(1);
    i8_wait<T::PIECES>(steps > 1);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    i8_fragments<T>(smem, 0, wn, wm, l31, half, w[0], a[0]);
    for (int s = 0; s < full; ++s) {
        const int8_t *st = smem + (s & 1) * T::STAGE, *next = smem + ((s + 1) & 1) * T::STAGE;
        i8_fragments<T>(st, 1, wn, wm, l31, half, w[1], a[1]);
        i8_multiply(w[0], a[0], acc);
        i8_fragments<T>(st, 2, wn, wm, l31, half, w[0], a[0]);
        i8_multiply(w[1], a[1], acc);
        i8_fragments<T>(st, 3, wn, wm, l31, half, w[1], a[1]);
        i8_multiply(w[0], a[0], acc);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (s + 2 < steps) issue(s + 2);
        i8_fragments<T>(next, 0, wn, wm, l31, half, w[0], a[0]);       // (behind the last step: not used)
        i8_multiply(w[1], a[1], acc);
    }
    if (tail) {          // only `left` codes of the last step belong to K; the other operand may hold anything behind them
        const int left = p.K - (steps_all - 1) * I8_BK;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            i8_fragments<T>(smem + (full & 1) * T::STAGE, kk, wn, wm, l31, half, w[0], a[0]);
#pragma unroll
            for (int j = 0; j < FM; ++j) a[0][j] = i8_mask(a[0][j], left - (2 * kk + half) * 16);
            i8_multiply(w[0], a[0], acc);
        }
    }
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int m = m0 + (wm * FM + j) * 32 + l31;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int n = n0 + (wn * FN + i) * 32 + 8 * g + 4 * half;
                const intx16& c = acc[i][j];
                if (p.partial == nullptr) i8_store4(p, m, n, c[4 * g], c[4 * g + 1], c[4 * g + 2], c[4 * g + 3]);
                else if (m < p.M) {
                    int* o = p.partial + ((size_t)blockIdx.y * p.M + m) * p.N + n;
#pragma unroll
                    for (int e = 0; e < 4; ++e) if (n + e < p.N) o[e] = c[4 * g + e];
                }
            }
        }
}

// the sums of a K that was split over several workgroups
__global__ void __launch_bounds__(256) gemm_i8_fold_kernel(const I8Problem p, int slices) {
    const int quads = (p.N + 3) / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)p.M * quads) return;
    const int m = (int)(i / quads), n = (int)(i % quads) * 4;
    int acc[4] = {0, 0, 0, 0};
    for (int s = 0; s < slices; ++s) {
        const int* o = p.partial + ((size_t)s * p.M + m) * p.N + n;
#pragma unroll
        for (int e = 0; e < 4; ++e) if (n + e < p.N) acc[e] += o[e];
    }
    i8_store4(p, m, n, acc[0], acc[1], acc[2], acc[3]);
}

// ------------------------------------------------------------------------------------------------------------------ choice
template <int WN, int WM, int FN, int FM>
static hipError_t launch_i8_tile(const I8Problem& p, int slices, hipStream_t s) {
    using T = I8Tile<WN, WM, FN, FM>;
    static const hipError_t prepared =
        hipFuncSetAttribute(reinterpret_cast<const void*>(&gemm_i8_kernel<WN, WM, FN, FM>), hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS);
    if (prepared != hipSuccess) return prepared;
    const int tiles = ((p.N + T::BN - 1) / T::BN) * ((p.M + T::BM - 1) / T::BM);
    hipLaunchKernelGGL((gemm_i8_kernel<WN, WM, FN, FM>), dim3(tiles, slices), dim3(T::THREADS), T::LDS, s, p);
    return hipGetLastError();
}

I8Plan gemm_i8_plan(int M, int N, int K) {
    I8Plan plan{};
    const int steps = (K + I8_BK - 1) / I8_BK;
    const int64_t t256 = (int64_t)((M + 255) / 256) * ((N + 255) / 256), t128 = (int64_t)((M + 127) / 128) * ((N + 127) / 128);
    const int64_t t64 = (int64_t)((M + 63) / 64) * ((N + 63) / 64);
    plan.slices = 1;
    if (t256 >= 192) plan.tile = 256;
    else if (t128 >= 192) plan.tile = 128;
    else {
        plan.tile = 64;
        int slices = (int)((384 + t64 - 1) / t64);
        slices = std::max(1, std::min(slices, steps / 4));
        plan.slices = slices;
    }
    plan.steps = (steps + plan.slices - 1) / plan.slices;
    plan.slices = (steps + plan.steps - 1) / plan.steps;
    return plan;
}

hipError_t launch_gemm_i8(I8Problem p, int* partial, hipStream_t s) {
    const I8Plan plan = gemm_i8_plan(p.M, p.N, p.K);
    p.steps = plan.steps;
    p.partial = plan.slices > 1 ? partial : nullptr;
    const size_t size = p.ytype == FBHIP_F32 ? 4 : 2;
    p.yvec = ((uintptr_t)p.y % (4 * size) == 0) && p.ldy % 4 == 0;
    hipError_t e;
    if (plan.tile == 256) e = launch_i8_tile<2, 4, 4, 2>(p, plan.slices, s);
    else if (plan.tile == 128) e = launch_i8_tile<2, 2, 2, 2>(p, plan.slices, s);
    else e = launch_i8_tile<2, 2, 1, 1>(p, plan.slices, s);
    if (e != hipSuccess || plan.slices == 1) return e;
    const int64_t quads = (int64_t)p.M * ((p.N + 3) / 4);
    hipLaunchKernelGGL(gemm_i8_fold_kernel, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, p, plan.slices);
    return hipGetLastError();
}

}  // namespace fbhip
