// One AdamW step over many tensors in one launch, moments in 32 or in 8 bits, and the global gradient norm that clips it.
//
//   g = gs * grad                          gs = grad_scale * min(1, max_norm / norm),  norm = |grad_scale| sqrt(sum of all grad^2)
//   m <- m + (1-b1)(g - m);   v <- b2 v + (1-b2) g g
//   p <- (1 - lr wd) p - lr/(1-b1^t) * m / (sqrt(v)/sqrt(1-b2^t) + eps)
//
// Bound by HBM: 28 bytes an element with fp32 parameters, gradients and moments, 16 with 8-bit moments.  Every stream is read once and
// written once; a lane holds eight consecutive elements, so that each 16-bit stream is one 16-byte access, an fp32 one two and a code
// stream one of 8 bytes, and a block of 256 elements that shares a scale is half a wave: its maximum is five lane exchanges.  (Four elements a
// lane leave room for more waves and take 20 % longer: the accesses are half as wide.)
// Measured, on a card whose large copy reaches 4.93 TB/s: 134 M fp32 parameters, bf16 gradients, 8-bit moments 407 us (4.64 TB/s, the arithmetic shows);
// 67 M in bf16 with fp32 moments and their norm 328 us (4.91 TB/s; more loads under way in the norm gained 1 % there and lost 10 % on 3.7 M); 3.7 M in
// fp32 21 us (32 bits), 23.5 us (8 bits 19, the norm 4 to 6), of which the start of a workgroup (scalars, tables, first loads) is a third.
// Root and quotient are correctly rounded, as the plain form's are.  With the instructions that are good to a step (v_sqrt_f32, v_rcp_f32) these took 376,
// 324, 21 and 21.7 us, but parameters differed in their last bit from the formulas' single-precision operations, and now and then a code of r by a step.
//
// 8-bit moments.  m and r = sqrt(v) are held as e4m3 codes times a power of two for each 256 elements (the least one under which the
// block's largest magnitude is at most 448).  r, not v: the step divides by sqrt(v), and the root halves the range that the codes have to
// span.  Codes are rounded up or down at random so that their mean is the value: a step moves v by a thousandth (1 - b2), half a code step
// is 3 %, and nearest rounding would never move r at all.  A positive r never rounds to zero (the update would divide by eps alone).
// The arithmetic before the codes is written without contraction and correctly rounded, so that a code depends on single-precision operations in the order
// of the formulas and on nothing else.  A value that is no number keeps its own code (NaN) and does not touch the block's scale.
#include "common.h"
#include "fbhip.h"

#include <cmath>

namespace fbhip {

constexpr int ADAMW_THREADS = 256, ADAMW_PER_LANE = 8, ADAMW_CHUNK = ADAMW_THREADS * ADAMW_PER_LANE;
static_assert(ADAMW_CHUNK == FBHIP_ADAMW_CHUNK, "the caller's chunk table counts chunks of this size");
constexpr int ADAMW_MAX_TENSORS = 384;       // gradient addresses travel in the kernel arguments (4 KB): valid in a captured graph
// Workgroups that are all on the 256 CUs at once and walk the chunks (more of them: the second lot runs on CUs that are half empty; with six a CU the
// walker networks take 28.0 us with 8-bit moments and clipping, with five 23.7).  With 32-bit moments three a CU keep memory busy, and more of them only
// spread the accesses: 67 M in bf16 329 us with three, 329 with four, 332 with five.  With 8-bit moments the arithmetic wants all five that the registers
// allow: 134 M 416 us, 470 with three, 431 with four, 463 with six.
constexpr int ADAMW_BLOCKS_32 = 3 * 256, ADAMW_BLOCKS_8 = 5 * 256;
constexpr int ADAMW_NORM_BLOCKS = 1024;      // one partial sum each, folded in order

// Workgroups count themselves off in 32 groups: 2048 additions to one address take 20 us, in turn, at the end of a step that takes 40.
constexpr int ADAMW_GROUPS = 32;

// The optimiser's scalars on the device (FBHIP_ADAMW_CONTROL_BYTES): a replayed graph advances them.
struct AdamwControl {
    int64_t t;                               // steps done
    double b1t, b2t;                         // b1^t, b2^t
    float norm;                              // of the gradients of the last step that clipped
    uint32_t root;                           // groups of workgroups that are done
    uint32_t pad[5];
    uint32_t group[ADAMW_GROUPS][16];        // workgroups that are done, on a line of their own for each group
};
static_assert(sizeof(AdamwControl) <= FBHIP_ADAMW_CONTROL_BYTES, "control block");

// The tables do not change while a kernel runs: scalar loads may read them.
template <class T>
__device__ __forceinline__ T table(const T* base, int i) {
#ifdef __HIP_DEVICE_COMPILE__
    return ((const T __attribute__((address_space(4)))*)(uintptr_t)base)[i];
#else
    return base[i];          // (the host pass has no such address space; it never runs this)
#endif
}

struct AdamwArgs {
    const fbhip_adamw_tensor* tensors;
    const int2* chunks;                      // (tensor, chunk of it)
    int first, last;                         // chunks of this launch
    int tensor0;                             // grad[] starts at this tensor
    int advance;                             // this launch is the step's last one
    int clip;
    AdamwControl* ctl;
    void *m, *v;                             // float, or codes
    float *m_scale, *r_scale;
    double lr, b1, b2;
    const float* lr_ptr;
    const double* partial;                   // of the gradients' squares
    int partials;
    float eps, grad_scale, max_norm;
    uint32_t seed;
    const void* grad[ADAMW_MAX_TENSORS];
    uint8_t gtype[ADAMW_MAX_TENSORS];
};
static_assert(sizeof(AdamwArgs) <= 4096, "kernel arguments");

struct NormArgs {
    const fbhip_adamw_tensor* tensors;
    const int2* chunks;
    int first, last, tensor0;
    double* partial;                         // one for each workgroup
    const void* grad[ADAMW_MAX_TENSORS];
    uint8_t gtype[ADAMW_MAX_TENSORS];
};
static_assert(sizeof(NormArgs) <= 4096, "kernel arguments");

__device__ __forceinline__ float bf16_float(uint32_t h) { return __uint_as_float(h << 16); }
__device__ __forceinline__ float fp16_float(uint16_t h) { _Float16 x; __builtin_memcpy(&x, &h, 2); return (float)x; }

__device__ __forceinline__ float load_one(const void* base, int64_t i, int type) {
    if (type == FBHIP_F32) return ((const float*)base)[i];
    const uint16_t h = ((const uint16_t*)base)[i];
    return type == FBHIP_BF16 ? bf16_float(h) : fp16_float(h);
}

// values side by side at any address: gfx950's global loads and stores need no alignment
typedef float floatx4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t uintx4_any __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ void load_eight(const void* base, int64_t i, int type, float (&x)[8]) {
    if (type == FBHIP_F32) {
        const floatx4_any a = *(const floatx4_any*)((const float*)base + i), b = *(const floatx4_any*)((const float*)base + i + 4);
        x[0] = a[0]; x[1] = a[1]; x[2] = a[2]; x[3] = a[3]; x[4] = b[0]; x[5] = b[1]; x[6] = b[2]; x[7] = b[3];
        return;
    }
    const uintx4_any w = *(const uintx4_any*)((const uint16_t*)base + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[2 * j] = type == FBHIP_BF16 ? bf16_float(w[j] & 0xFFFFu) : fp16_float((uint16_t)w[j]);
        x[2 * j + 1] = type == FBHIP_BF16 ? __uint_as_float(w[j] & 0xFFFF0000u) : fp16_float((uint16_t)(w[j] >> 16));
    }
}

// Where element i of a tensor lies: dense tensors are one run in storage order; a row-strided matrix has its own leading dimension.
struct Walk {
    int64_t row; int col, cols, ld;
    __device__ __forceinline__ Walk(int64_t i, int cols_, int ld_) : cols(cols_), ld(ld_) { row = i / cols_; col = (int)(i - row * cols_); }
    __device__ __forceinline__ int64_t at() const { return row * ld + col; }
    __device__ __forceinline__ void next() { if (++col == cols) { col = 0; ++row; } }
};

// The gradient's eight elements from i on (zero behind the tensor's end).
__device__ __forceinline__ void load_grad(const fbhip_adamw_tensor& T, const void* g, int gtype, int64_t i, float (&x)[8]) {
    const bool flat = T.cols == 0 || (gtype & FBHIP_GRAD_DENSE);
    gtype &= FBHIP_GRAD_DENSE - 1;
    if (flat && i + 8 <= T.numel) { load_eight(g, i, gtype, x); return; }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 0.f;
    if (i >= T.numel) return;
    if (flat) {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (i + j < T.numel) x[j] = load_one(g, i + j, gtype);
    } else {
        Walk w(i, T.cols, T.ld);
#pragma unroll
        for (int j = 0; j < 8; ++j) { if (i + j < T.numel) x[j] = load_one(g, w.at(), gtype); w.next(); }
    }
}

// A 32-bit word for an element: its place is multiplied and shifted into the step's key (two rounds of multiply and shift-xor: the published 32-bit
// finaliser of MurmurHash3).
__device__ __forceinline__ uint32_t finish_word(uint32_t h) {
    h = (h ^ (h >> 16)) * 0x85EBCA6Bu;
    h = (h ^ (h >> 13)) * 0xC2B2AE35u;
    return h ^ (h >> 16);
}
// of the eight elements from place i on; places beyond 2^32 take a key of their own (i is a multiple of eight: none of them crosses over)
__device__ __forceinline__ void element_words(int64_t i, uint32_t key, uint32_t (&w)[8]) {
    const uint32_t first = (uint32_t)i * 0x9E3779B1u + key + (uint32_t)((uint64_t)i >> 32) * 0x27D4EB2Fu;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) w[j] = finish_word(first + j * 0x9E3779B1u);
}

// e4m3 codes of eight lane values and the block's scale (half a wave = 256 elements); u: 16 random bits for each value
template <bool POSITIVE>
__device__ __forceinline__ uint2 encode_eight(const float (&x)[8], const uint32_t (&u)[8], float& scale) {
    uint32_t mag[8], top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        mag[j] = __float_as_uint(x[j]) & 0x7FFFFFFFu;
        top = max(top, mag[j]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    const bool odd = top >= 0x7F800000u;          // somewhere in the block something is no number: it does not count for the scale
    if (odd) {
        top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, mag[j] < 0x7F800000u ? mag[j] : 0u);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    }
    // 448 = 1.75 * 2^8: the exponent field of 2^k with top * 2^-k <= 448; at least 1, so that 2^k and 2^-k are normal numbers
    const int field = max((int)((top + 0x1FFFFFu) >> 23) - 8, 1);
    scale = __uint_as_float((uint32_t)field << 23);
    const float inv = __uint_as_float((uint32_t)(254 - field) << 23);
    uint32_t c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float y = __uint_as_float(mag[j]) * inv;
        // three mantissa bits stay; below 2^-6 the codes are evenly spaced, which adding 2^-6 brings about
        const bool small = y < 0.015625f;
        const uint32_t z = __float_as_uint(small ? y + 0.015625f : y);
        c[j] = ((u[j] << 4) + z - (small ? 968u << 20 : 960u << 20)) >> 20;
        if (POSITIVE) c[j] = max(c[j], min(mag[j], 1u));
        else c[j] |= (__float_as_uint(x[j]) >> 24) & 0x80u;
    }
    if (odd) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (mag[j] >= 0x7F800000u) c[j] = 0x7Fu | (POSITIVE ? 0u : (__float_as_uint(x[j]) >> 24) & 0x80u);
    }
    return make_uint2(c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24);
}

__device__ __forceinline__ void decode_eight(uint2 q, float scale, float (&x)[8]) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, true);
    const auto c = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, true);
    x[0] = a[0] * scale; x[1] = a[1] * scale; x[2] = b[0] * scale; x[3] = b[1] * scale;
    x[4] = c[0] * scale; x[5] = c[1] * scale; x[6] = d[0] * scale; x[7] = d[1] * scale;
}

// lanes and waves folded in a fixed order
__device__ __forceinline__ double block_sum(double x, double* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

template <int BITS>
__global__ void __launch_bounds__(ADAMW_THREADS, 5) adamw_kernel(const AdamwArgs a) {
#pragma clang fp contract(off)
    __shared__ double red[4], shared_lr, shared_ibc1;
    __shared__ float shared_rbc2, shared_gs;
    __shared__ uint32_t shared_key;
    const int tid = threadIdx.x;
    float norm = 0.f;
    if (a.clip) {
        // every workgroup adds the partial sums for itself, in the same order
        double x = 0.0;
        for (int k = tid; k < a.partials; k += ADAMW_THREADS) x += a.partial[k];
        norm = (float)(fabs((double)a.grad_scale) * sqrt(block_sum(x, red)));
        if (blockIdx.x == 0 && tid == 0 && a.advance) a.ctl->norm = norm;
        if (!(norm < __uint_as_float(0x7F800000u))) return;          // not a number: nothing changes, nothing counts
    }
    if (tid == 0) {
        const double b1t = a.ctl->b1t * a.b1, b2t = a.ctl->b2t * a.b2;
        shared_lr = a.lr_ptr != nullptr ? (double)*a.lr_ptr : a.lr;
        shared_ibc1 = 1.0 / (1.0 - b1t);
        shared_rbc2 = (float)(1.0 / sqrt(1.0 - b2t));
        shared_gs = a.grad_scale * (norm > a.max_norm ? a.max_norm / norm : 1.f);
        shared_key = finish_word(a.seed ^ (uint32_t)(a.ctl->t + 1) * 0x27D4EB2Fu);
    }
    __syncthreads();
    const float gs = shared_gs, rbc2 = shared_rbc2, eps = a.eps;
    const double lr = shared_lr, ibc1 = shared_ibc1;
    const uint32_t key = shared_key;
    const float w1 = (float)(1.0 - a.b1), w2 = (float)(1.0 - a.b2), b2 = (float)a.b2;
    for (int c = a.first + (int)blockIdx.x; c < a.last; c += (int)gridDim.x) {
        const int2 e = table(a.chunks, c);
        const fbhip_adamw_tensor T = table(a.tensors, e.x);
        const int64_t i = (int64_t)e.y * ADAMW_CHUNK + tid * ADAMW_PER_LANE;
        // the moments are padded to whole blocks of 256 for each tensor: half a wave is inside or outside as one
        if (i >= ((T.numel + 255) & ~(int64_t)255)) continue;
        const int64_t s = T.at + i;
        float g[8], p[8], m[8], v[8];
        load_grad(T, a.grad[e.x - a.tensor0], a.gtype[e.x - a.tensor0], i, g);
        const bool whole = T.cols == 0 && i + 8 <= T.numel;
        if (whole) load_eight(T.p, i, T.dtype, p);
        else {
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = 0.f;
            if (T.cols == 0) {
#pragma unroll
                for (int j = 0; j < 8; ++j) if (i + j < T.numel) p[j] = load_one(T.p, i + j, T.dtype);
            } else {
                Walk w(i, T.cols, T.ld);
#pragma unroll
                for (int j = 0; j < 8; ++j) { if (i + j < T.numel) p[j] = load_one(T.p, w.at(), T.dtype); w.next(); }
            }
        }
        if (BITS == 32) {
            load_eight(a.m, s, FBHIP_F32, m);
            load_eight(a.v, s, FBHIP_F32, v);
        } else {
            const uint2 qm = *(const uint2*)((const uint8_t*)a.m + s), qr = *(const uint2*)((const uint8_t*)a.v + s);
            decode_eight(qm, a.m_scale[s >> 8], m);
            decode_eight(qr, a.r_scale[s >> 8], v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = v[j] * v[j];
        }
        const double lrt = lr * T.lr_scale;
        const float keep = (float)(1.0 - lrt * T.weight_decay), ss = (float)(lrt * ibc1);
        float r[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float gr = g[j] * gs;
            m[j] = m[j] + w1 * (gr - m[j]);
            v[j] = v[j] * b2 + (w2 * gr) * gr;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            r[j] = sqrtf(v[j]);
            p[j] = p[j] * keep - ss * (m[j] / (r[j] * rbc2 + eps));
        }
        uint32_t word[8];
        if (BITS == 8 || T.dtype == FBHIP_BF16) element_words(s, key, word);
        if (BITS == 32) {
            *(float4*)((float*)a.m + s) = make_float4(m[0], m[1], m[2], m[3]);
            *(float4*)((float*)a.m + s + 4) = make_float4(m[4], m[5], m[6], m[7]);
            *(float4*)((float*)a.v + s) = make_float4(v[0], v[1], v[2], v[3]);
            *(float4*)((float*)a.v + s + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t u[8];
            float scale;
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = word[j] >> 16;
            *(uint2*)((uint8_t*)a.m + s) = encode_eight<false>(m, u, scale);
            if ((tid & 31) == 0) a.m_scale[s >> 8] = scale;
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = word[j] & 0xFFFFu;
            *(uint2*)((uint8_t*)a.v + s) = encode_eight<true>(r, u, scale);
            if ((tid & 31) == 0) a.r_scale[s >> 8] = scale;
        }
        if (T.dtype == FBHIP_BF16) {
            // up or down at random: bf16 steps are 0.4 % apart, and an update of a thousandth of that still has to count on average
            uint32_t h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t b = __float_as_uint(p[j]);
                h[j] = p[j] != p[j] ? 0x7FC0u : (b + (word[j] * 0x9E3779B1u >> 16)) >> 16;
            }
            if (whole) {
                *(uintx4_any*)((uint16_t*)T.p + i) = uintx4_any{h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16};
            } else if (i < T.numel) {
                Walk w(i, T.cols == 0 ? 0x7FFFFFFF : T.cols, T.ld);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (i + j < T.numel) ((uint16_t*)T.p)[T.cols == 0 ? i + j : w.at()] = (uint16_t)h[j];
                    w.next();
                }
            }
        } else if (whole) {
            *(floatx4_any*)((float*)T.p + i) = floatx4_any{p[0], p[1], p[2], p[3]};
            *(floatx4_any*)((float*)T.p + i + 4) = floatx4_any{p[4], p[5], p[6], p[7]};
        } else if (i < T.numel) {
            Walk w(i, T.cols == 0 ? 0x7FFFFFFF : T.cols, T.ld);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (i + j < T.numel) ((float*)T.p)[T.cols == 0 ? i + j : w.at()] = p[j];
                w.next();
            }
        }
    }
    if (tid != 0 || !a.advance) return;
    // every workgroup has read the scalars when the last one comes here: it moves them to the next step
    const uint32_t mine = blockIdx.x % ADAMW_GROUPS, members = (gridDim.x - mine + ADAMW_GROUPS - 1) / ADAMW_GROUPS;
    if (__hip_atomic_fetch_add(&a.ctl->group[mine][0], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != members - 1) return;
    a.ctl->group[mine][0] = 0;
    const uint32_t groups = gridDim.x < ADAMW_GROUPS ? gridDim.x : ADAMW_GROUPS;
    if (__hip_atomic_fetch_add(&a.ctl->root, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != groups - 1) return;
    a.ctl->root = 0;
    a.ctl->t += 1;
    a.ctl->b1t *= a.b1;
    a.ctl->b2t *= a.b2;
}

// The squares are summed in doubles: the square of the largest fp32 is far inside their range.
__global__ void __launch_bounds__(ADAMW_THREADS) adamw_norm_kernel(const NormArgs a) {
    __shared__ double red[4];
    double acc = 0.0;
    for (int c = a.first + (int)blockIdx.x; c < a.last; c += (int)gridDim.x) {
        const int2 e = table(a.chunks, c);
        const fbhip_adamw_tensor T = table(a.tensors, e.x);
        float g[8];
        load_grad(T, a.grad[e.x - a.tensor0], a.gtype[e.x - a.tensor0], (int64_t)e.y * ADAMW_CHUNK + (int)threadIdx.x * ADAMW_PER_LANE, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc += (double)g[j] * (double)g[j];
    }
    const double sum = block_sum(acc, red);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = sum;
}

__global__ void adamw_set_kernel(AdamwControl* c, int64_t t, double b1t, double b2t) {
    c->t = t; c->b1t = b1t; c->b2t = b2t;
    c->norm = 0.f;
    c->root = 0;
    for (int g = 0; g < ADAMW_GROUPS; ++g) c->group[g][0] = 0;
}

hipError_t launch_adamw_set(void* control, int64_t t, double b1, double b2, hipStream_t s) {
    hipLaunchKernelGGL(adamw_set_kernel, dim3(1), dim3(1), 0, s, (AdamwControl*)control, t, std::pow(b1, (double)t), std::pow(b2, (double)t));
    return hipGetLastError();
}

hipError_t launch_adamw_step(const fbhip_adamw* o, const void* const* grads, const uint8_t* gtypes, const float* lr_ptr, double lr,
                             float grad_scale, int clip, float max_norm, hipStream_t s) {
    const int n = o->n_tensors, launches = (n + ADAMW_MAX_TENSORS - 1) / ADAMW_MAX_TENSORS;
    int partials = 0;
    if (clip) {
        NormArgs a{};
        a.tensors = o->tensors; a.chunks = (const int2*)o->chunks;
        for (int l = 0; l < launches; ++l) {
            const int t0 = l * ADAMW_MAX_TENSORS, t1 = min(n, t0 + ADAMW_MAX_TENSORS);
            a.first = o->host_first_chunk[t0]; a.last = o->host_first_chunk[t1]; a.tensor0 = t0;
            for (int t = t0; t < t1; ++t) { a.grad[t - t0] = grads[t]; a.gtype[t - t0] = gtypes[t]; }
            const int blocks = max(1, min(ADAMW_NORM_BLOCKS, a.last - a.first));
            a.partial = o->partials + partials;
            partials += blocks;
            hipLaunchKernelGGL(adamw_norm_kernel, dim3(blocks), dim3(ADAMW_THREADS), 0, s, a);
        }
    }
    AdamwArgs a{};
    a.tensors = o->tensors; a.chunks = (const int2*)o->chunks; a.ctl = (AdamwControl*)o->control; a.clip = clip;
    a.partial = o->partials; a.partials = partials; a.max_norm = max_norm;
    a.m = o->m; a.v = o->v; a.m_scale = o->m_scale; a.r_scale = o->r_scale;
    a.lr = lr; a.lr_ptr = lr_ptr; a.b1 = o->beta1; a.b2 = o->beta2; a.eps = o->eps; a.grad_scale = grad_scale; a.seed = o->seed;
    for (int l = 0; l < launches; ++l) {
        const int t0 = l * ADAMW_MAX_TENSORS, t1 = min(n, t0 + ADAMW_MAX_TENSORS);
        a.first = o->host_first_chunk[t0]; a.last = o->host_first_chunk[t1]; a.tensor0 = t0;
        a.advance = l == launches - 1;
        for (int t = t0; t < t1; ++t) { a.grad[t - t0] = grads[t]; a.gtype[t - t0] = gtypes[t]; }
        const int blocks = max(1, min(o->bits == 32 ? ADAMW_BLOCKS_32 : ADAMW_BLOCKS_8, a.last - a.first));
        if (o->bits == 32) hipLaunchKernelGGL(adamw_kernel<32>, dim3(blocks), dim3(ADAMW_THREADS), 0, s, a);
        else hipLaunchKernelGGL(adamw_kernel<8>, dim3(blocks), dim3(ADAMW_THREADS), 0, s, a);
    }
    return hipGetLastError();
}

int adamw_partials(int n_tensors) { return (n_tensors + ADAMW_MAX_TENSORS - 1) / ADAMW_MAX_TENSORS * ADAMW_NORM_BLOCKS; }

}  // namespace fbhip

