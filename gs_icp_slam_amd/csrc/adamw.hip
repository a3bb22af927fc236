// The AdamW step over many tensors in one launch, its moments held in 32 bits or in 8, and the global gradient norm that clips it.
//
//   g' = c g,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2,  p = (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Pure streaming: with f32 parameters 28 bytes per element (7 accesses of 4) with 32-bit moments and 16 with 8-bit ones, against ~35 and ~85 VALU
// instructions.  The file is compiled without contraction of a * b + c, so that the moments round like the written formulas and the codes of the 8-bit
// moments can be predicted bit for bit.
//
// 8-BIT MOMENTS.  Two bytes per element and two per block of 128 consecutive elements of a tensor.  A code c > 0 with the block's base exponent b stands for
// (1 + (c & 7) / 8) * 2^((c >> 3) + b - 127) — as f32 bits simply (c << 20) + (b << 23) —, c = 0 for zero.  First moment: sign and 7 bits (16 exponents),
// second: 8 bits (32 exponents); the base is the exponent of the block's largest finite value less 14 or 30 (at least 1), so the largest always has a code, with
// room for one carry.  Why a floating code with a shared POWER OF TWO: Adam divides by sqrt(v), so what counts is the relative error of small values too, and
// the block's scale costs no multiplication and no division.  Why STOCHASTIC rounding: with b2 = 0.999 one step moves v by a thousandth of itself, and codes are
// 6 to 12 % apart — rounded to nearest, v would never move unless the gradient jumped eightfold; rounded up with the probability of the distance to the code
// below, its expectation is exact.  Second moments above zero never round to zero (the smallest code instead): the denominator must not vanish; first moments below the
// smallest code keep their expectation (that code with probability |m| / code, else zero).  As 2 * 15 exponents of v cover the same gradients as 14 of m, an element
// at either floor still moves by at most twice the block's largest step.  Values that are not finite stay so in their own element: magnitude 127 is NaN,
// second-moment code 255 is infinity.
// The random bits are a function of (seed, step, place of the tensor in the list, element): one hashed word per 8 elements, times an odd constant per element — its
// high and low half are the 16 bits of v and m (each uniform, because an odd multiplier permutes the words).
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <utility>
#include <vector>

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "../../include/gsicp_hip.h"
#include "raster_common.hpp"

namespace gsicp {
extern thread_local std::string g_last_error;

namespace {

constexpr int TABLE = 40;             // tensors per launch: the table travels in the kernel arguments (< 4 KB), nothing is copied or kept
constexpr int NORM_TABLE = 64;
constexpr int TILE_ELEMS = 2048;      // elements per workgroup and pass: 256 lanes x 8
constexpr int STEP_GRID = 2048;       // workgroups of a large launch (8 per CU)
constexpr int NORM_GRID = 2048;       // partial sums of one norm launch
constexpr int NORM_SMALL_TILES = 128; // 4 KB tiles that one workgroup of 16 waves takes by itself
constexpr int QBLOCK = 128;           // elements per base exponent: 16 lanes x 8

enum Dtype { F32 = 0, BF16 = 1, F16 = 2 };

// vector types without an alignment demand beyond the element's: views of a flat buffer begin anywhere
typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(2)));

struct StepEntry {
    void* p;
    const void* g;
    void* s0;              // exp_avg, or the packed 8-bit moments
    void* s1;              // exp_avg_sq, or the base exponents
    float* master;
    long long numel;
    double lr, wd;
    int row_width;         // elements per map row (live rows, masks); 0: whole tensor
    uint16_t kind;         // Dtype | 4 with a master
    uint16_t frozen;       // rows with a non-zero freeze word are left alone
    int src, place;        // index in the caller's arrays (device learning rates), place in the list (random bits)
};
struct StepTable {
    uint32_t first[64];    // first tile of each tensor; ~0 behind the last: a wave finds the tensor of a tile by one ballot
    StepEntry e[TABLE];
};
struct StepHyper {
    float b1, omb1, b2, omb2, eps;
    float inv_bc2_sqrt;    // 1 / sqrt(1 - b2^t)            (host step count)
    double inv_bc1;        // 1 / (1 - b1^t)
    double db1, db2;       // for the same on the device     (device step count)
    const float* clip;     // device: the factor of every gradient (NULL: 1)
    const double* lr_dev;
    const int* step_dev;
    int step;              // host: the step count; device: what to add to *step_dev
    uint32_t seed, tiles;
    const uint32_t* guard_count;
    uint32_t guard_limit;
    const int *live_rows, *row_freeze, *grad_rows;
};
static_assert(sizeof(StepTable) + sizeof(StepHyper) <= 4096, "kernel arguments of a launch");

__device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x7FEB352Du;
    x = (x ^ (x >> 15)) * 0x846CA68Bu;
    return x ^ (x >> 16);
}
__device__ __forceinline__ uint32_t lane_word(int e) {
    constexpr uint32_t w[8] = {0x6A09E667u, 0xBB67AE85u, 0x3C6EF373u, 0xA54FF53Bu, 0x510E527Fu, 0x9B05688Du, 0x1F83D9ABu, 0x5BE0CD19u};
    return w[e];
}

// the tensor a tile belongs to: lane l compares the tile with tensor l's first one
__device__ __forceinline__ int find_tensor(const uint32_t* first, uint32_t tile) {
    return __popcll(__ballot(first[threadIdx.x & 63] <= tile)) - 1;
}

__device__ __forceinline__ float from16(uint32_t h, int dtype) {
    return dtype == BF16 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half((unsigned short)h));
}
__device__ __forceinline__ uint32_t to16(float x, int dtype) {        // round to nearest, ties to even
    if (dtype == F16) return __half_as_ushort(__float2half_rn(x));
    const uint32_t b = __float_as_uint(x);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return (b >> 16) | 0x40u;    // NaN stays NaN
    return (b + 0x7FFFu + ((b >> 16) & 1u)) >> 16;
}

// eight consecutive elements; FULL: all of them exist, else only the first nv
template <int DT, bool FULL>
__device__ __forceinline__ void load8(const void* base, long long at, int nv, float out[8]) {
    if (DT == F32) {
        const float* p = (const float*)base + at;
        if (FULL) {
            const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) { out[j] = a[j]; out[j + 4] = b[j]; }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) out[j] = j < nv ? p[j] : 0.f;
        }
    } else {
        const uint16_t* p = (const uint16_t*)base + at;
        if (FULL) {
            const u32x4 a = *(const u32x4*)p;
#pragma unroll
            for (int j = 0; j < 8; ++j) out[j] = from16((a[j >> 1] >> (16 * (j & 1))) & 0xFFFFu, DT);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) out[j] = j < nv ? from16(p[j], DT) : 0.f;
        }
    }
}
template <int DT, bool FULL>
__device__ __forceinline__ void store8(void* base, long long at, int nv, const float x[8]) {
    if (DT == F32) {
        float* p = (float*)base + at;
        if (FULL) {
            f32x4 a, b;
#pragma unroll
            for (int j = 0; j < 4; ++j) { a[j] = x[j]; b[j] = x[j + 4]; }
            *(f32x4*)p = a;
            *(f32x4*)(p + 4) = b;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) if (j < nv) p[j] = x[j];
        }
    } else {
        uint16_t* p = (uint16_t*)base + at;
        if (FULL) {
            u32x4 a;
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] = to16(x[2 * j], DT) | (to16(x[2 * j + 1], DT) << 16);
            *(u32x4*)p = a;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) if (j < nv) p[j] = (uint16_t)to16(x[j], DT);
        }
    }
}
template <bool FULL>
__device__ __forceinline__ void load_codes(const void* base, long long at, int nv, uint32_t c[4]) {
    const uint16_t* p = (const uint16_t*)base + at;
    if (FULL) {
        const u32x4 a = *(const u32x4*)p;
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = a[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = (2 * j < nv ? (uint32_t)p[2 * j] : 0u) | (2 * j + 1 < nv ? (uint32_t)p[2 * j + 1] << 16 : 0u);
    }
}
template <bool FULL>
__device__ __forceinline__ void store_codes(void* base, long long at, int nv, const uint32_t c[4]) {
    uint16_t* p = (uint16_t*)base + at;
    if (FULL) {
        u32x4 a;
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = c[j];
        *(u32x4*)p = a;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (j < nv) p[j] = (uint16_t)(c[j >> 1] >> (16 * (j & 1)));
    }
}

__device__ __forceinline__ float decode_m(uint32_t c16, uint32_t bm23) {
    const uint32_t mag = c16 & 0x7Fu;
    const uint32_t bits = ((mag << 20) + bm23) | ((c16 & 0x80u) << 24);
    return mag == 0u ? 0.f : __uint_as_float(mag == 127u ? 0x7FC00000u : bits);
}
__device__ __forceinline__ float decode_v(uint32_t c16, uint32_t bv23) {
    const uint32_t c = (c16 >> 8) & 0xFFu;
    return c == 0u ? 0.f : __uint_as_float(c == 255u ? 0x7F800000u : (c << 20) + bv23);
}
// largest value of the 16 lanes of a row, in every one of them: four rotations
__device__ __forceinline__ uint32_t row16_max(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xF, 0xF, true));   // row_ror:8
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xF, 0xF, true));   // row_ror:4
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xF, 0xF, true));   // row_ror:2
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xF, 0xF, true));   // row_ror:1
    return x;
}
__device__ __forceinline__ uint32_t base_exponent(uint32_t top, int below) {
    const int b = (int)(top >> 23) - below;
    return (uint32_t)(b < 1 ? 1 : b);
}

// what one step needs to know of a tensor, after the hyper-parameters are folded
struct Fold { float b1, omb1, b2, omb2, eps, ibc2, decay, step_size, clip; };

__device__ __forceinline__ void adamw(float& p, float& m, float& v, float g, const Fold& f) {
    m = m * f.b1 + g * f.omb1;
    v = v * f.b2 + g * f.omb2 * g;
    p = p * f.decay;
    p = p - f.step_size * (m / (sqrtf(v) * f.ibc2 + f.eps));
}

template <bool Q8, int DT, bool MASTER, bool FULL, bool MASKED>
__device__ __forceinline__ void step_tile(const StepEntry& e, const Fold& f, const int* row_freeze, const int* grad_rows, uint32_t key, uint32_t tile, long long numel) {
    const long long at = (long long)tile * TILE_ELEMS + 8 * threadIdx.x;
    const int nv = FULL ? 8 : (int)max(0ll, min(8ll, numel - at));
    float p[8], g[8], m[8], v[8];
    uint32_t c[4], exps = 0;
    if (MASTER) load8<F32, FULL>(e.master, at, nv, p); else load8<DT, FULL>(e.p, at, nv, p);
    load8<DT, FULL>(e.g, at, nv, g);
    const long long block = (long long)tile * (TILE_ELEMS / QBLOCK) + (threadIdx.x >> 4);
    if (Q8) {
        load_codes<FULL>(e.s0, at, nv, c);
        if (FULL || nv > 0) exps = ((const uint16_t*)e.s1)[block];
    } else {
        load8<F32, FULL>(e.s0, at, nv, m);
        load8<F32, FULL>(e.s1, at, nv, v);
    }
    uint32_t keep = 0;                          // elements of frozen rows
    if (MASKED) {
        const uint32_t w = (uint32_t)e.row_width;
        if (w && nv > 0) {
            uint32_t row = (uint32_t)at / w, col = (uint32_t)at - row * w;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (FULL || j < nv) {
                    if (grad_rows && grad_rows[row] <= 0) g[j] = 0.f;     // whatever the gradient's memory holds there
                    if (e.frozen && row_freeze[row] != 0) keep |= 1u << j;
                }
                if (++col == w) { col = 0; ++row; }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] *= f.clip;
    if (Q8) {
        const uint32_t bm23 = (exps & 0xFFu) << 23, bv23 = (exps >> 8) << 23;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t c16 = c[j >> 1] >> (16 * (j & 1));
            m[j] = decode_m(c16, bm23);
            v[j] = decode_v(c16, bv23);
        }
    }
    float p0[8], m0[8], v0[8];
    if (MASKED && !Q8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) { p0[j] = p[j]; m0[j] = m[j]; v0[j] = v[j]; }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) adamw(p[j], m[j], v[j], g[j], f);
    if (MASKED && !Q8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (keep >> j & 1u) { p[j] = p0[j]; m[j] = m0[j]; v[j] = v0[j]; }
    }
    if (MASTER) store8<F32, FULL>(e.master, at, nv, p);
    store8<DT, FULL>(e.p, at, nv, p);
    if (!Q8) {
        store8<F32, FULL>(e.s0, at, nv, m);
        store8<F32, FULL>(e.s1, at, nv, v);
        return;
    }
    uint32_t tm = 0, tv = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t mb = __float_as_uint(m[j]) & 0x7FFFFFFFu, vb = __float_as_uint(v[j]) & 0x7FFFFFFFu;
        if (FULL || j < nv) {
            tm = max(tm, mb < 0x7F800000u ? mb : 0u);
            tv = max(tv, vb < 0x7F800000u ? vb : 0u);
        }
    }
    const uint32_t bm = base_exponent(row16_max(tm), 14), bv = base_exponent(row16_max(tv), 30);
    const float low = __uint_as_float((bm << 23) + (1u << 20)), low16 = low * 0x1p-16f;
    const uint32_t word = mix32(((uint32_t)tile * (TILE_ELEMS / 8) + threadIdx.x) ^ key);
    uint32_t o[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t r = word * lane_word(j), um = r & 0xFFFFu, uv = r >> 16;
        const uint32_t mb = __float_as_uint(m[j]) & 0x7FFFFFFFu, vb = __float_as_uint(v[j]) & 0x7FFFFFFFu;
        const float a = __uint_as_float(mb);
        uint32_t mc = ((mb + (um << 4) + 8u) >> 20) - (bm << 3);
        if (a < low) mc = a > low16 * ((float)um + 0.5f) ? 1u : 0u;
        if (mc != 0u) mc |= __float_as_uint(m[j]) >> 31 << 7;
        if (mb >= 0x7F800000u) mc = 127u;
        int vs = (int)((vb + (uv << 4) + 8u) >> 20) - (int)(bv << 3);
        uint32_t vc = vb == 0u ? 0u : (uint32_t)(vs < 1 ? 1 : vs);
        if (vb >= 0x7F800000u) vc = 255u;
        o[j >> 1] |= (mc | vc << 8) << (16 * (j & 1));
    }
    store_codes<FULL>(e.s0, at, nv, o);
    if ((threadIdx.x & 15) == 0 && (FULL || nv > 0)) ((uint16_t*)e.s1)[block] = (uint16_t)(bm | bv << 8);
}

// One launch: grid-stride over the tiles of up to 40 tensors.  DEV: step count and learning rates come from device memory (a captured graph replays them).
template <bool Q8, bool DEV, bool MASKED>
__global__ __launch_bounds__(256) void adamw_step_kernel(StepTable t, StepHyper h) {
    double inv_bc1 = h.inv_bc1;
    float ibc2 = h.inv_bc2_sqrt;
    int step = h.step;
    if (DEV) {
        if (h.guard_count && *h.guard_count > h.guard_limit) return;      // the iteration that made these gradients is void: nothing moves
        __shared__ double s_bc1;
        __shared__ float s_bc2;
        step += *h.step_dev;
        if (threadIdx.x == 0) {
            s_bc1 = 1.0 / (1.0 - pow(h.db1, (double)step));
            s_bc2 = (float)(1.0 / sqrt(1.0 - pow(h.db2, (double)step)));
        }
        __syncthreads();
        inv_bc1 = s_bc1;
        ibc2 = s_bc2;
    }
    const float clip = h.clip ? *h.clip : 1.f;
    for (uint32_t tile = blockIdx.x; tile < h.tiles; tile += gridDim.x) {
        const int k = __builtin_amdgcn_readfirstlane(find_tensor(t.first, tile));
        const StepEntry& e = t.e[k];
        const uint32_t mine = tile - t.first[k];
        long long numel = e.numel;
        if (DEV && h.live_rows && e.row_width > 0) numel = min(numel, (long long)*h.live_rows * e.row_width);   // rows behind the live count are not parameters
        const long long left = numel - (long long)mine * TILE_ELEMS;
        if (left <= 0) continue;
        const double lr = DEV ? h.lr_dev[e.src] : e.lr;
        const Fold f = {h.b1, h.omb1, h.b2, h.omb2, h.eps, ibc2, (float)(1.0 - lr * e.wd), (float)(lr * inv_bc1), clip};
        const uint32_t key = Q8 ? mix32(h.seed + (uint32_t)step * 0x9E3779B1u + (uint32_t)e.place * 0x85EBCA6Bu) : 0u;
        const bool full = left >= TILE_ELEMS;
#define GSICP_STEP(DT, MASTER)                                                                                                             \
    (full ? step_tile<Q8, DT, MASTER, true, MASKED>(e, f, h.row_freeze, h.grad_rows, key, mine, numel)                                      \
          : step_tile<Q8, DT, MASTER, false, MASKED>(e, f, h.row_freeze, h.grad_rows, key, mine, numel))
        if (MASKED || e.kind == F32) GSICP_STEP(F32, false);
        else if (e.kind == BF16) GSICP_STEP(BF16, false);
        else if (e.kind == F16) GSICP_STEP(F16, false);
        else if (e.kind == (BF16 | 4)) GSICP_STEP(BF16, true);
        else GSICP_STEP(F16, true);
#undef GSICP_STEP
    }
}

__global__ void adamw_bump_kernel(int* step_dev, const uint32_t* guard_count, uint32_t guard_limit, uint32_t* skipped) {
    if (guard_count && *guard_count > guard_limit) {
        if (skipped) *skipped += 1u;
        return;
    }
    *step_dev += 1;
}

// ------------------------------------------------------------------------------------------------ values of the codes
struct DecodeEntry { const void* codes; const void* exps; void* m; void* v; long long numel; };
struct DecodeTable { uint32_t first[64]; DecodeEntry e[64]; };

template <int DT, bool FULL>
__device__ __forceinline__ void decode_tile(const DecodeEntry& e, uint32_t tile) {
    const long long at = (long long)tile * TILE_ELEMS + 8 * threadIdx.x;
    const int nv = FULL ? 8 : (int)max(0ll, min(8ll, e.numel - at));
    if (nv == 0) return;
    uint32_t c[4];
    load_codes<FULL>(e.codes, at, nv, c);
    const uint32_t exps = ((const uint16_t*)e.exps)[at / QBLOCK];
    float m[8], v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t c16 = c[j >> 1] >> (16 * (j & 1));
        m[j] = decode_m(c16, (exps & 0xFFu) << 23);
        v[j] = decode_v(c16, (exps >> 8) << 23);
    }
    store8<DT, FULL>(e.m, at, nv, m);
    store8<DT, FULL>(e.v, at, nv, v);
}
// bf16 holds every code's value exactly (four significant bits, f32's exponents)
template <int DT>
__global__ __launch_bounds__(256) void adamw_decode_kernel(DecodeTable t, uint32_t tiles) {
    for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int k = __builtin_amdgcn_readfirstlane(find_tensor(t.first, tile));
        const DecodeEntry& e = t.e[k];
        const uint32_t mine = tile - t.first[k];
        if (e.numel - (long long)mine * TILE_ELEMS >= TILE_ELEMS) decode_tile<DT, true>(e, mine);
        else decode_tile<DT, false>(e, mine);
    }
}

// ------------------------------------------------------------------------------------------------ global norm
// Squares and sums in 64 bits: 133 M f16 gradients summed in 32 would lose what the clip factor needs to be the same from run to run and split to split, and the squares of large
// or small f32 gradients would leave its range.  The sums are split over the workgroups by position alone and joined in a fixed order.
struct NormEntry { const void* g; long long numel; int dtype, pad; };
struct NormTable { uint32_t first[64]; NormEntry e[NORM_TABLE]; };

__host__ __device__ constexpr int norm_tile_elems(int dtype, int bytes) { return bytes / (dtype == F32 ? 4 : 2); }

template <int DT>
__device__ __forceinline__ double square_sum16(const u32x4& r) {      // of one 16-byte load
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (DT == F32) { const double x = __uint_as_float(r[j]); s = __builtin_fma(x, x, s); }
        else {
            const double x = from16(r[j] & 0xFFFFu, DT), y = from16(r[j] >> 16, DT);
            s = __builtin_fma(x, x, s);
            s = __builtin_fma(y, y, s);
        }
    }
    return s;
}
// `lanes` lanes, four 16-byte loads of each in flight; lane l of load k takes unit k * lanes + l
template <int DT>
__device__ __forceinline__ double norm_tile(const NormEntry& e, uint32_t tile, int lanes, int lane) {
    constexpr int V = DT == F32 ? 4 : 8;
    const long long at = (long long)tile * (4 * V * lanes), left = e.numel - at;
    const char* p = (const char*)e.g + at * (16 / V);
    double s = 0.0;
    if (left >= 4 * V * lanes) {
        u32x4 r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = *(const u32x4*)(p + 16 * (size_t)(k * lanes + lane));
#pragma unroll
        for (int k = 0; k < 4; ++k) s += square_sum16<DT>(r[k]);
    } else {
        for (int k = 0; k < 4; ++k) {
            const long long u = (long long)(k * lanes + lane) * V;
            if (u + V <= left) s += square_sum16<DT>(*(const u32x4*)(p + u * (16 / V)));
            else
                for (long long j = u; j < left && j < u + V; ++j) {
                    const double x = DT == F32 ? ((const float*)p)[j] : from16(((const uint16_t*)p)[j], DT);
                    s = __builtin_fma(x, x, s);
                }
        }
    }
    return s;
}
__device__ __forceinline__ double norm_any_tile(const NormTable& t, uint32_t tile, int lanes, int lane) {
    const int k = __builtin_amdgcn_readfirstlane(find_tensor(t.first, tile));
    const NormEntry& e = t.e[k];
    const uint32_t mine = tile - t.first[k];
    return e.dtype == F32 ? norm_tile<F32>(e, mine, lanes, lane) : e.dtype == BF16 ? norm_tile<BF16>(e, mine, lanes, lane) : norm_tile<F16>(e, mine, lanes, lane);
}
template <int WAVES>
__device__ __forceinline__ double block_sum(double s) {      // complete in thread 0
    __shared__ double part[WAVES];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_down(s, off, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = part[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += part[w];
    }
    return s;
}
// the norm, and min(1, max_norm / (norm + 1e-6)): NaN when the norm is, as torch.nn.utils.clip_grad_norm_ has it
__device__ __forceinline__ void norm_results(double sum, double max_norm, float* norm_out, float* clip_out) {
    const float norm = (float)sqrt(sum);
    const double c = max_norm / ((double)norm + 1e-6);
    *norm_out = norm;
    if (clip_out) *clip_out = max_norm > 0.0 ? (float)(c > 1.0 ? 1.0 : c) : 1.f;
}
__global__ __launch_bounds__(256) void grad_norm_kernel(NormTable t, uint32_t tiles, double* partial) {
    double s = 0.0;
    for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) s += norm_any_tile(t, tile, 256, threadIdx.x);
    s = block_sum<4>(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}
__global__ __launch_bounds__(1024) void grad_norm_finish_kernel(const double* __restrict__ partial, int n, double max_norm, float* norm_out, float* clip_out) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) s += partial[i];
    s = block_sum<16>(s);
    if (threadIdx.x == 0) norm_results(s, max_norm, norm_out, clip_out);
}
// few small tensors: one workgroup, a tile per WAVE, no second launch
__global__ __launch_bounds__(1024) void grad_norm_small_kernel(NormTable t, uint32_t tiles, double max_norm, float* norm_out, float* clip_out) {
    double s = 0.0;
    for (uint32_t tile = threadIdx.x >> 6; tile < tiles; tile += 16) s += norm_any_tile(t, tile, 64, threadIdx.x & 63);
    s = block_sum<16>(s);
    if (threadIdx.x == 0) norm_results(s, max_norm, norm_out, clip_out);
}

// ------------------------------------------------------------------------------------------------ host
int fail(const char* what) { g_last_error = what; return -2; }

size_t dtype_bytes(int dt) { return dt == F32 ? 4 : 2; }

// what a call writes must not overlap: a tensor given twice would be updated by two workgroups at once
bool disjoint(std::vector<std::pair<uintptr_t, uintptr_t>>& r) {
    if (!std::is_sorted(r.begin(), r.end())) std::sort(r.begin(), r.end());
    for (size_t i = 1; i < r.size(); ++i) if (r[i].first < r[i - 1].second) return false;
    return true;
}

uint32_t tiles_of(long long numel) { return (uint32_t)((numel + TILE_ELEMS - 1) / TILE_ELEMS); }

struct StepCall {
    int n; void* const* params; const void* const* grads; float* const* masters; void* const* s0; void* const* s1;
    const long long* numel; const int* dtype; const double* lr; const double* wd; const int* place;
};

template <bool Q8>
void launch_step(dim3 grid, bool dev, bool masked, hipStream_t stream, const StepTable& t, const StepHyper& h) {
    if (!dev) hipLaunchKernelGGL((adamw_step_kernel<Q8, false, false>), grid, dim3(256), 0, stream, t, h);
    else if (!masked) hipLaunchKernelGGL((adamw_step_kernel<Q8, true, false>), grid, dim3(256), 0, stream, t, h);
    else hipLaunchKernelGGL((adamw_step_kernel<Q8, true, true>), grid, dim3(256), 0, stream, t, h);
}

template <bool Q8>
int adamw_call(const StepCall& c, double b1, double b2, double eps, int step, uint32_t seed, const float* clip, const gsicp_adamw_device* dev, hipStream_t stream) {
    if (c.n < 0 || (c.n > 0 && (!c.params || !c.grads || !c.s0 || !c.s1 || !c.numel || !c.dtype || !c.wd))) return fail("gsicp_adamw_step: missing arrays");
    if (!(b1 >= 0.0 && b1 < 1.0 && b2 >= 0.0 && b2 < 1.0 && eps >= 0.0)) return fail("gsicp_adamw_step: betas are in [0, 1), eps is not negative");
    if (dev) {
        if (!dev->lr_dev || !dev->step_dev || dev->bump_step < 0 || dev->bump_step > 2)
            return fail("gsicp_adamw_step: the device form needs learning rates, a step counter and bump_step 0, 1 or 2");
        if ((dev->live_rows || dev->row_freeze || dev->grad_rows) && !dev->row_width) return fail("gsicp_adamw_step: live rows and row masks need row_width");
        if (dev->row_freeze && !dev->group_frozen) return fail("gsicp_adamw_step: row_freeze needs group_frozen");
        if (Q8 && (dev->live_rows || dev->row_freeze)) return fail("gsicp_adamw_step_8bit: live rows and frozen rows would share block exponents with rows that move");
    } else if (step < 1 || (c.n > 0 && !c.lr)) {
        return fail("gsicp_adamw_step: the host form needs learning rates and a step count of at least 1");
    }
    const bool masked = dev && (dev->row_freeze || dev->grad_rows);
    static thread_local std::vector<std::pair<uintptr_t, uintptr_t>> ranges;
    ranges.clear();
    for (int k = 0; k < c.n; ++k) {
        const long long n = c.numel[k];
        if (n < 0 || n >= (1ll << 35)) return fail("gsicp_adamw_step: a tensor has 0 to 2^35 - 1 elements");
        if (n == 0) continue;
        const int dt = c.dtype[k];
        if (dt < F32 || dt > F16) return fail("gsicp_adamw_step: dtype is 0 (f32), 1 (bf16) or 2 (f16)");
        float* master = c.masters ? c.masters[k] : nullptr;
        if (!c.params[k] || !c.grads[k] || !c.s0[k] || !c.s1[k]) return fail("gsicp_adamw_step: null pointer of a tensor that is not empty");
        if (master && dt == F32) return fail("gsicp_adamw_step: an f32 parameter has no master");
        if (masked && (dt != F32 || n >= (1ll << 32))) return fail("gsicp_adamw_step: row masks go with f32 parameters of less than 2^32 elements");
        auto add = [&](const void* q, size_t bytes) { ranges.emplace_back((uintptr_t)q, (uintptr_t)q + bytes); };
        add(c.params[k], (size_t)n * dtype_bytes(dt));
        if (master) add(master, (size_t)n * 4);
        if (Q8) { add(c.s0[k], (size_t)n * 2); add(c.s1[k], (size_t)((n + QBLOCK - 1) / QBLOCK) * 2); }
        else { add(c.s0[k], (size_t)n * 4); add(c.s1[k], (size_t)n * 4); }
    }
    if (!disjoint(ranges)) return fail("gsicp_adamw_step: two tensors that the step writes overlap (the same one given twice?)");

    StepHyper h = {};
    h.b1 = (float)b1; h.omb1 = (float)(1.0 - b1); h.b2 = (float)b2; h.omb2 = (float)(1.0 - b2); h.eps = (float)eps;
    h.db1 = b1; h.db2 = b2; h.clip = clip; h.seed = seed;
    if (dev) {
        h.lr_dev = dev->lr_dev; h.step_dev = dev->step_dev; h.step = dev->bump_step == 2 ? 0 : 1;
        h.guard_count = dev->guard_count; h.guard_limit = dev->guard_limit;
        h.live_rows = dev->live_rows; h.row_freeze = dev->row_freeze; h.grad_rows = dev->grad_rows;
    } else {
        h.step = step;
        h.inv_bc1 = 1.0 / (1.0 - std::pow(b1, step));
        h.inv_bc2_sqrt = (float)(1.0 / std::sqrt(1.0 - std::pow(b2, step)));
    }
    {
        ProfileScope ps(ST_ADAM, stream);
        for (int k = 0; k < c.n;) {
            StepTable t = {};
            int n = 0;
            unsigned long long tiles = 0;
            for (; k < c.n && n < TABLE; ++k) {
                if (c.numel[k] == 0) continue;
                StepEntry& e = t.e[n];
                e.p = c.params[k]; e.g = c.grads[k]; e.s0 = c.s0[k]; e.s1 = c.s1[k]; e.master = c.masters ? c.masters[k] : nullptr;
                e.numel = c.numel[k]; e.lr = c.lr ? c.lr[k] : 0.0; e.wd = c.wd[k];
                e.row_width = dev && dev->row_width ? dev->row_width[k] : 0;
                e.kind = (uint16_t)(c.dtype[k] | (e.master ? 4 : 0));
                e.frozen = (uint16_t)(dev && dev->row_freeze && dev->group_frozen[k] && e.row_width > 0);
                e.src = k; e.place = c.place ? c.place[k] : k;
                t.first[n++] = (uint32_t)tiles;
                tiles += tiles_of(e.numel);
                if (tiles > 0xF0000000ull) return fail("gsicp_adamw_step: too many elements in one call");
            }
            for (int i = n; i < 64; ++i) t.first[i] = 0xFFFFFFFFu;
            if (n == 0) break;
            h.tiles = (uint32_t)tiles;
            launch_step<Q8>(dim3((unsigned)std::min<unsigned long long>(tiles, STEP_GRID)), dev != nullptr, masked, stream, t, h);
        }
        if (dev && dev->bump_step == 1)
            hipLaunchKernelGGL(adamw_bump_kernel, dim3(1), dim3(1), 0, stream, dev->step_dev, dev->guard_count, dev->guard_limit, dev->skipped);
    }
    if (hipGetLastError() != hipSuccess) { g_last_error = "gsicp_adamw_step: kernel launch failed"; return -1; }
    return 0;
}

}  // namespace
}  // namespace gsicp

using namespace gsicp;

extern "C" {

int gsicp_adamw_step(int n, void* const* params, const void* const* grads, float* const* masters, float* const* exp_avg, float* const* exp_avg_sq,
                     const long long* numel, const int* dtype, const double* lr, const double* weight_decay, double beta1, double beta2, double eps, int step,
                     const float* clip, const gsicp_adamw_device* dev, void* stream) {
    try {
        return adamw_call<false>({n, params, grads, masters, (void* const*)exp_avg, (void* const*)exp_avg_sq, numel, dtype, lr, weight_decay, nullptr}, beta1, beta2, eps, step, 0u,
                                 clip, dev, (hipStream_t)stream);
    } catch (const std::exception& ex) { g_last_error = ex.what(); return -1; }
}

int gsicp_adamw_step_8bit(int n, void* const* params, const void* const* grads, float* const* masters, uint16_t* const* moments, uint16_t* const* block_exps,
                          const long long* numel, const int* dtype, const double* lr, const double* weight_decay, double beta1, double beta2, double eps, int step,
                          uint32_t seed, const int* place, const float* clip, const gsicp_adamw_device* dev, void* stream) {
    try {
        return adamw_call<true>({n, params, grads, masters, (void* const*)moments, (void* const*)block_exps, numel, dtype, lr, weight_decay, place}, beta1, beta2, eps, step, seed,
                                clip, dev, (hipStream_t)stream);
    } catch (const std::exception& ex) { g_last_error = ex.what(); return -1; }
}

int gsicp_adamw_decode(int n, const uint16_t* const* moments, const uint16_t* const* block_exps, void* const* exp_avg, void* const* exp_avg_sq, const long long* numel,
                       int dtype, void* stream_v) {
    hipStream_t stream = (hipStream_t)stream_v;
    if (n < 0 || (n > 0 && (!moments || !block_exps || !exp_avg || !exp_avg_sq || !numel))) return fail("gsicp_adamw_decode: missing arrays");
    if (dtype != F32 && dtype != BF16) return fail("gsicp_adamw_decode: dtype is 0 (f32) or 1 (bf16)");
    for (int k = 0; k < n; ++k) {
        if (numel[k] < 0 || numel[k] >= (1ll << 35)) return fail("gsicp_adamw_decode: a tensor has 0 to 2^35 - 1 elements");
        if (numel[k] > 0 && (!moments[k] || !block_exps[k] || !exp_avg[k] || !exp_avg_sq[k])) return fail("gsicp_adamw_decode: null pointer of a tensor that is not empty");
    }
    for (int k = 0; k < n;) {
        DecodeTable t = {};
        int m = 0;
        unsigned long long tiles = 0;
        for (; k < n && m < 64; ++k) {
            if (numel[k] == 0) continue;
            t.e[m] = {moments[k], block_exps[k], exp_avg[k], exp_avg_sq[k], numel[k]};
            t.first[m++] = (uint32_t)tiles;
            tiles += tiles_of(numel[k]);
            if (tiles > 0xF0000000ull) return fail("gsicp_adamw_decode: too many elements in one call");
        }
        for (int i = m; i < 64; ++i) t.first[i] = 0xFFFFFFFFu;
        if (m == 0) break;
        const dim3 grid((unsigned)std::min<unsigned long long>(tiles, STEP_GRID));
        if (dtype == F32) hipLaunchKernelGGL((adamw_decode_kernel<F32>), grid, dim3(256), 0, stream, t, (uint32_t)tiles);
        else hipLaunchKernelGGL((adamw_decode_kernel<BF16>), grid, dim3(256), 0, stream, t, (uint32_t)tiles);
    }
    if (hipGetLastError() != hipSuccess) { g_last_error = "gsicp_adamw_decode: kernel launch failed"; return -1; }
    return 0;
}

size_t gsicp_grad_norm_scratch_bytes(int n) { return n <= 0 ? 8 : (size_t)((n + NORM_TABLE - 1) / NORM_TABLE) * NORM_GRID * sizeof(double); }

int gsicp_grad_norm(int n, const void* const* grads, const long long* numel, const int* dtype, double max_norm, float* norm_out, float* clip_out, void* scratch,
                    void* stream_v) {
    hipStream_t stream = (hipStream_t)stream_v;
    if (n < 0 || (n > 0 && (!grads || !numel || !dtype)) || !norm_out || !scratch) return fail("gsicp_grad_norm: missing arrays");
    unsigned long long small = 0;
    int used_tensors = 0;
    for (int k = 0; k < n; ++k) {
        if (numel[k] < 0 || numel[k] >= (1ll << 35)) return fail("gsicp_grad_norm: a tensor has 0 to 2^35 - 1 elements");
        if (numel[k] == 0) continue;
        if (!grads[k] || dtype[k] < F32 || dtype[k] > F16) return fail("gsicp_grad_norm: null pointer, or a dtype that is not 0 (f32), 1 (bf16) or 2 (f16)");
        ++used_tensors;
        const int te = norm_tile_elems(dtype[k], 64 * 64);
        small += (unsigned long long)((numel[k] + te - 1) / te);
    }
    const bool one = used_tensors <= NORM_TABLE && small <= NORM_SMALL_TILES;
    const int tile_bytes = one ? 64 * 64 : 256 * 64;
    double* partial = (double*)scratch;
    int used = 0;
    for (int k = 0; k < n || one;) {
        NormTable t = {};
        int m = 0;
        unsigned long long tiles = 0;
        for (; k < n && m < NORM_TABLE; ++k) {
            if (numel[k] == 0) continue;
            t.e[m] = {grads[k], numel[k], dtype[k], 0};
            t.first[m++] = (uint32_t)tiles;
            const int te = norm_tile_elems(dtype[k], tile_bytes);
            tiles += (unsigned long long)((numel[k] + te - 1) / te);
            if (tiles > 0xF0000000ull) return fail("gsicp_grad_norm: too many elements in one call");
        }
        for (int i = m; i < 64; ++i) t.first[i] = 0xFFFFFFFFu;
        if (one) {
            hipLaunchKernelGGL(grad_norm_small_kernel, dim3(1), dim3(1024), 0, stream, t, (uint32_t)tiles, max_norm, norm_out, clip_out);
            break;
        }
        if (m == 0) break;
        const unsigned grid = (unsigned)std::min<unsigned long long>(tiles, NORM_GRID);
        hipLaunchKernelGGL(grad_norm_kernel, dim3(grid), dim3(256), 0, stream, t, (uint32_t)tiles, partial + used);
        used += (int)grid;
    }
    if (!one) hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(1024), 0, stream, (const double*)partial, used, max_norm, norm_out, clip_out);
    if (hipGetLastError() != hipSuccess) { g_last_error = "gsicp_grad_norm: kernel launch failed"; return -1; }
    return 0;
}

}  // extern "C"
