// tlg_rows.h -- elements, rows and waves of the operators over rows of logits
// (tlg_vocab.hip, tlg_verify.hip), and what their entries ask of the rows.
#pragma once
#include "tlg_internal.h"
#include "../../include/tltrain.h"
#include <math.h>

// ------------------------------------------------------------- elements --
// Rows are read and written 16 bytes at a time, on the 16-byte grid of the
// address space: a row that starts `sh` elements behind a grid point takes
// `nv` grid vectors, of which the first and the last may hold elements of its
// neighbours; those are loaded and stored element by element.
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
template <int TYPE> struct El {
    static constexpr int VE = TYPE == TLG_F32 ? 4 : 8;              // elements of a vector
    static constexpr int SZ = TYPE == TLG_F32 ? 4 : 2;
    static constexpr unsigned NEG = TYPE == TLG_F32 ? 0xff800000u : TYPE == TLG_F16 ? 0xfc00u : 0xff80u;  // -inf
};

template <int TYPE> __device__ __forceinline__ float el_float(unsigned bits)
{
    if constexpr (TYPE == TLG_F32) return __uint_as_float(bits);
    else if constexpr (TYPE == TLG_F16) return (float)__builtin_bit_cast(_Float16, (unsigned short)bits);
    else return __uint_as_float(bits << 16);
}
// Between two uses of a vector kept in registers: without it the compiler keeps
// the elements unpacked from the first use to the second, twice the registers.
__device__ __forceinline__ void keep_packed(u32x4 &r) { asm volatile("" : "+v"(r)); }
// element e of a raw vector; e is a constant where it is called
template <int TYPE> __device__ __forceinline__ float el_at(const u32x4 &r, int e)
{
    if constexpr (TYPE == TLG_F32) return __uint_as_float(r[e]);
    else if constexpr (TYPE == TLG_BF16) return __uint_as_float(e & 1 ? r[e >> 1] & 0xffff0000u : r[e >> 1] << 16);
    else return el_float<TYPE>(e & 1 ? r[e >> 1] >> 16 : r[e >> 1] & 0xffffu);
}
template <int TYPE> __device__ __forceinline__ unsigned el_bits(float v)      // rounded to nearest even
{
    if constexpr (TYPE == TLG_F32) return __float_as_uint(v);
    else if constexpr (TYPE == TLG_F16) return __builtin_bit_cast(unsigned short, (_Float16)v);
    else return __builtin_bit_cast(unsigned short, (__bf16)v);
}
template <int TYPE> __device__ __forceinline__ float el_load(const char *x, int i)
{
    if constexpr (TYPE == TLG_F32) return ((const float *)x)[i];
    else return el_float<TYPE>(((const unsigned short *)x)[i]);
}
template <int TYPE> __device__ __forceinline__ void el_store(char *x, int i, float v)
{
    if constexpr (TYPE == TLG_F32) ((float *)x)[i] = v;
    else ((unsigned short *)x)[i] = (unsigned short)el_bits<TYPE>(v);
}

template <int TYPE> struct Row {
    static constexpr int VE = El<TYPE>::VE;
    const char *x;              // element 0
    const u32x4 *v;             // grid vector 0
    int V, sh, nv, f0, f1;      // whole vectors: [f0, f1)
    __device__ __forceinline__ Row(const void *base, long long ld, size_t r, int V_)
    {
        x = (const char *)base + (long long)r * ld * El<TYPE>::SZ;
        const int a = (int)((uintptr_t)x & 15);
        v = (const u32x4 *)(x - a);
        V = V_;
        sh = a / El<TYPE>::SZ;
        nv = (V + sh + VE - 1) / VE;
        f0 = sh ? 1 : 0;
        f1 = (V + sh) / VE;
    }
    __device__ __forceinline__ u32x4 edge(int j) const
    {
        u32x4 r;
        unsigned b[VE];
#pragma unroll
        for (int e = 0; e < VE; e++) {
            const int i = j * VE + e - sh;
            b[e] = El<TYPE>::NEG;
            if (i >= 0 && i < V) {
                if constexpr (TYPE == TLG_F32) b[e] = ((const unsigned *)x)[i];
                else b[e] = ((const unsigned short *)x)[i];
            }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if constexpr (TYPE == TLG_F32) r[k] = b[k];
            else r[k] = b[2 * k] | b[2 * k + 1] << 16;
        }
        return r;
    }
    // vector j, -inf where it is no part of the row
    __device__ __forceinline__ u32x4 any(int j) const
    {
        if (j >= f0 && j < f1) return v[j];
        if (j >= nv) {
            const unsigned n = TYPE == TLG_F32 ? El<TYPE>::NEG : El<TYPE>::NEG * 0x10001u;
            return u32x4{n, n, n, n};
        }
        return edge(j);
    }
};

// ------------------------------------------------------------ threads of a row --
// W waves work on one row: 64 W threads, synchronised by a barrier or, for one
// wave, by its own order.
template <int W> __device__ __forceinline__ void row_sync()
{
    if constexpr (W > 1) __syncthreads();
    else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}
// Sum and maximum over a wave in a fixed order: neighbours in each row of 16
// lanes by data-parallel moves, then the four rows; every lane of an active
// wave must take part, and every lane gets the result.
template <int CTRL> __device__ __forceinline__ float lane_move(float v)
{
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float row_of(float v, int r)
{
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 16 * r));
}
#define WAVE_REDUCE(name, OP)                                                              \
    __device__ __forceinline__ float name(float v)                                         \
    {                                                                                      \
        v = OP(v, lane_move<0xB1>(v));      /* quad_perm 1,0,3,2 */                         \
        v = OP(v, lane_move<0x4E>(v));      /* quad_perm 2,3,0,1 */                         \
        v = OP(v, lane_move<0x141>(v));     /* row_half_mirror */                          \
        v = OP(v, lane_move<0x140>(v));     /* row_mirror */                               \
        return OP(OP(row_of(v, 0), row_of(v, 1)), OP(row_of(v, 2), row_of(v, 3)));         \
    }
__device__ __forceinline__ float add_op(float a, float b) { return a + b; }
WAVE_REDUCE(wave_max, fmaxf)
WAVE_REDUCE(wave_sum, add_op)

// scale (x - m); halves where the difference of finite values passes fp32 and
// its product need not
__device__ __forceinline__ float lp_scaled(float x, float m, float scale)
{
    const float d = x - m;
    return d > -INFINITY || x == -INFINITY ? d * scale : (0.5f * x - 0.5f * m) * scale * 2.f;
}

// -------------------------------------------------------------------- checks --
static inline size_t vb_size(int type) { return type == TLG_F32 ? 4 : 2; }

// what every entry asks of its logits; `who` names the entry in the error
static inline int vb_check(const char *who, const void *logits, int type, long long ld, int N, int V)
{
    if (type != TLG_F32 && type != TLG_F16 && type != TLG_BF16) return tlg_fail(TLG_EINVAL, "%s: type %d", who, type);
    if (N < 0 || N > TLG_VOCAB_ROWS || V <= 0 || V > TLG_VOCAB_MAX || ld < V)
        return tlg_fail(TLG_EINVAL, "%s: N=%d V=%d ld=%lld", who, N, V, ld);
    if (N > 0 && (!logits || (uintptr_t)logits % vb_size(type)))
        return tlg_fail(TLG_EINVAL, "%s: logits %p", who, logits);
    return TLG_OK;
}
static inline int vb_check_ws(const char *who, const void *ws, size_t have, size_t need)
{
    if (need && (have < need || !ws || (uintptr_t)ws % 16))
        return tlg_fail(TLG_EINVAL, "%s: workspace %p of %zu bytes, %zu needed", who, ws, have, need);
    return TLG_OK;
}
// a scale or temperature: its multiples by log2 e and back must be finite and normal
static inline bool vb_positive(float s) { return s >= 1e-30f && s <= 1e30f; }
