// sam3_lora_amd -- row operators of include/sam3_seq_amd.h (gfx950): RMS norm with the residual's addition and an 8-bit output,
// rotary positions with several axes.  Both move each byte once and are bound by HBM; what they compute rides along.
#include "seq_common.inc"

#include "sam3_fp8_amd.h"
#include "sam3_seq_amd.h"

using namespace seq;

namespace {
thread_local char g_err[256] = "";
}

int sam3_seq_fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}
void sam3_seq_clear_error() { g_err[0] = 0; }

namespace {

// ------------------------------------------------------------------------------------------------------------ RMS norm
// h = x + r,  rstd = 1 / sqrt(mean(h^2) + eps),  y = h rstd w.
// LPR lanes hold a row (8 .. 64: a part of a wave, several rows side by side for narrow norms such as one over a head; 256: the
// whole workgroup, for rows that one wave's registers do not hold), CPL chunks of 8 elements per lane, in registers between
// the sum and the output: each byte moves once.  The weight stays in registers over the rows that a workgroup walks.
// y and the 8-bit image come from the unrounded fp32 h; only what leaves is rounded.
struct NormFwd {
    const void *x, *r, *w;
    void *y, *h;
    unsigned short* low;
    float* rstd;
    unsigned char* q8;
    float* scales;
    long long ldx, ldr, M;
    int C, group;       // group: log2 of the columns that share a scale, 0: the whole row
    float eps, fmax;
};

// sum over the LPR lanes of a row; the workgroup's version goes through LDS
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* lds) {
    if (LPR <= 64) return lane_sum<LPR < 64 ? LPR : 64>(v);
    v = lane_sum<64>(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (lds[0] + lds[1]) + (lds[2] + lds[3]);
    __syncthreads();
    return v;
}
// magnitudes as their bit patterns: they order like the numbers, and a NaN is above all of them
__device__ __forceinline__ unsigned mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ unsigned lane_max(unsigned v, int lanes) {
    for (int o = lanes / 2; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o, 64));
    return v;
}
template <int LPR>
__device__ __forceinline__ unsigned row_max(unsigned v, unsigned* lds) {
    v = lane_max(v, LPR < 64 ? LPR : 64);
    if (LPR <= 64) return v;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = max(max(lds[0], lds[1]), max(lds[2], lds[3]));
    __syncthreads();
    return v;
}

template <int FMT>
__device__ __forceinline__ unsigned to_fp8x4(float a, float b, float c, float d) {
    int w = 0;
    if (FMT == SAM3_FP8_E4M3) {
        w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    } else {
        w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, w, false);
        w = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true);
    }
    return (unsigned)w;
}

// What the rounding of h to 16 bits took away, to about a tenth of it, in two bits: 0, or +-3/8 of the last place that is left (the
// difference of the bit patterns counts in last places whatever the exponent).  The weight's gradient sums products with h over the rows:
// with the rounded h it is off by sqrt(2) of its own rounding, and worse by chance; with these bits by 1.05.  A sixteenth of y's bytes.
__device__ __forceinline__ unsigned low_bits(const float* h, const Raw8<bf16_t>& o) {
    const unsigned b[4] = {o.a.x, o.a.y, o.a.z, o.a.w};
    unsigned code = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int d = (int)(__float_as_uint(h[j]) - (j & 1 ? b[j / 2] & 0xffff0000u : b[j / 2] << 16));
        code |= (d > 0x3000 ? 1u : d < -0x3000 ? 3u : 0u) << (2 * j);
    }
    return code;
}
__device__ __forceinline__ void add_low_bits(float* h, unsigned code) {
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = __uint_as_float(__float_as_uint(h[j]) + ((int)(code << (30 - 2 * j)) >> 30) * 0x6000);
}
__device__ __forceinline__ unsigned low_bits(const float*, const Raw8<float>&) { return 0; }

// Q8: 0 none, 1 e4m3, 2 e5m2
template <typename T, int LPR, int CPL, int Q8>
__global__ __launch_bounds__(256) void k_rms_fwd(NormFwd a) {
    __shared__ float lds[4];
    constexpr int RPB = 256 / LPR;      // rows of a workgroup at a time
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const T *x = (const T*)a.x, *r = (const T*)a.r;
    Raw8<T> w[CPL];
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
        const int c = (i * LPR + lane) * 8;
        if (c < a.C) w[i].load((const T*)a.w + c);
    }
    for (long long row0 = (long long)blockIdx.x * RPB; row0 < a.M; row0 += (long long)gridDim.x * RPB) {
        const long long row = row0 + sub;
        const bool live = row < a.M;
        float h[CPL][8];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < CPL; ++i) {
            const int c = (i * LPR + lane) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = 0.f;
            if (live && c < a.C) {
                Raw8<T> v;
                v.load(x + row * a.ldx + c);
                v.get(h[i]);
                if (r) {
                    float t[8];
                    v.load(r + row * a.ldr + c);
                    v.get(t);
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[i][j] += t[j];
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) s += h[i][j] * h[i][j];
            }
        }
        const float rs = rsqrtf(row_sum<LPR>(s, lds) / (float)a.C + a.eps);
        if (live && lane == 0 && a.rstd) a.rstd[row] = rs;
#pragma unroll
        for (int i = 0; i < CPL; ++i) {
            const int c = (i * LPR + lane) * 8;
            if (live && c < a.C) {
                Raw8<T> o;
                if (a.h) {
                    o.set(h[i]);
                    o.store((T*)a.h + row * a.C + c);
                    if (sizeof(T) == 2 && a.low) a.low[(row * a.C + c) >> 3] = (unsigned short)low_bits(h[i], o);
                }
                float g[8];
                w[i].get(g);
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] = h[i][j] * rs * g[j];
                if (a.y) {
                    o.set(h[i]);
                    o.store((T*)a.y + row * a.C + c);
                }
            }
        }
        if (Q8) {
            unsigned m[CPL];
#pragma unroll
            for (int i = 0; i < CPL; ++i) {
                m[i] = 0u;
#pragma unroll
                for (int j = 0; j < 8; ++j) m[i] = max(m[i], mag(h[i][j]));
            }
            if (a.group) {              // a group is group / 8 neighbouring lanes of one chunk row
#pragma unroll
                for (int i = 0; i < CPL; ++i) m[i] = lane_max(m[i], 1 << (a.group - 3));
            } else {
#pragma unroll
                for (int i = 1; i < CPL; ++i) m[0] = max(m[0], m[i]);
                m[0] = row_max<LPR>(m[0], reinterpret_cast<unsigned*>(lds));
#pragma unroll
                for (int i = 1; i < CPL; ++i) m[i] = m[0];
            }
#pragma unroll
            for (int i = 0; i < CPL; ++i) {
                const int c = (i * LPR + lane) * 8;
                // (an infinity in y makes the scale infinite and the image NaN: the group is lost either way)
                const float am = __uint_as_float(max(m[i], 0x33800000u)), inv = a.fmax / am;
                if (live && c < a.C) {
                    constexpr int F = Q8 == 1 ? SAM3_FP8_E4M3 : SAM3_FP8_E5M2;
                    *reinterpret_cast<uint2*>(a.q8 + row * a.C + c) =
                        make_uint2(to_fp8x4<F>(h[i][0] * inv, h[i][1] * inv, h[i][2] * inv, h[i][3] * inv),
                                   to_fp8x4<F>(h[i][4] * inv, h[i][5] * inv, h[i][6] * inv, h[i][7] * inv));
                    if (a.group ? (c & ((1 << a.group) - 1)) == 0 : c == 0)
                        a.scales[a.group ? row * (a.C >> a.group) + (c >> a.group) : row] = am / a.fmax;
                }
            }
        }
    }
}

struct NormBwd {
    const void *gy, *gh, *h, *w;
    const unsigned short* low;
    const float* rstd;
    void* gx;
    float* part;        // [workgroups, C] fp32, or NULL: no weight gradient
    long long ldh, M;
    int C;
};

// gx = rstd (u - xhat mean(u xhat)) + gh,  u = gy w,  xhat = h rstd.  A workgroup walks rows gridDim apart and keeps its part of
// gw = sum gy xhat in registers; its rows' parts meet in LDS in a fixed order and leave as one row of partial sums.
template <typename T, int LPR, int CPL>
__global__ __launch_bounds__(256) void k_rms_bwd(NormBwd a) {
    __shared__ float lds[4];
    __shared__ float comb[256 * 8];     // one chunk row of every row's part of the weight gradient
    constexpr int RPB = 256 / LPR;
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const T *gy = (const T*)a.gy, *gh = (const T*)a.gh, *hh = (const T*)a.h;
    Raw8<T> w[CPL];
    float acc[CPL][8];
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
        const int c = (i * LPR + lane) * 8;
        if (c < a.C) w[i].load((const T*)a.w + c);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = 0.f;
    }
    for (long long row0 = (long long)blockIdx.x * RPB; row0 < a.M; row0 += (long long)gridDim.x * RPB) {
        const long long row = row0 + sub;
        const bool live = row < a.M;
        const float rs = live ? a.rstd[row] : 0.f;
        float u[CPL][8], xh[CPL][8];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < CPL; ++i) {
            const int c = (i * LPR + lane) * 8;
            if (live && c < a.C) {
                Raw8<T> v, g;
                v.load(hh + row * a.ldh + c);
                g.load(gy + row * a.C + c);
                v.get(xh[i]);
                if (sizeof(T) == 2 && a.low) add_low_bits(xh[i], a.low[(row * a.C + c) >> 3]);
                g.get(u[i]);
                float wv[8];
                w[i].get(wv);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    xh[i][j] *= rs;
                    acc[i][j] += u[i][j] * xh[i][j];
                    u[i][j] *= wv[j];
                    s += u[i][j] * xh[i][j];
                }
            }
        }
        const float mean = row_sum<LPR>(s, lds) / (float)a.C;
        if (a.gx) {
#pragma unroll
            for (int i = 0; i < CPL; ++i) {
                const int c = (i * LPR + lane) * 8;
                if (live && c < a.C) {
                    Raw8<T> o;
                    float t[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                    if (gh) {
                        o.load(gh + row * a.C + c);
                        o.get(t);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) t[j] += rs * (u[i][j] - xh[i][j] * mean);
                    o.set(t);
                    o.store((T*)a.gx + row * a.C + c);
                }
            }
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
        const int c0 = i * LPR * 8, c = c0 + lane * 8;
        if (RPB > 1) {
#pragma unroll
            for (int j = 0; j < 8; ++j) comb[(sub * LPR + lane) * 8 + j] = acc[i][j];
            __syncthreads();
            for (int k = threadIdx.x; k < LPR * 8; k += 256)
                if (c0 + k < a.C) {
                    float v = 0.f;
                    for (int t = 0; t < RPB; ++t) v += comb[t * LPR * 8 + k];
                    a.part[(long long)blockIdx.x * a.C + c0 + k] = v;
                }
            __syncthreads();
        } else if (c < a.C) {
#pragma unroll
            for (int j = 0; j < 8; ++j) a.part[(long long)blockIdx.x * a.C + c + j] = acc[i][j];
        }
    }
}

// gw[c] = sum of n partial rows, 32 columns x 32 row groups per workgroup, fixed order
template <typename T>
__global__ __launch_bounds__(1024) void k_rms_gw(const float* __restrict__ part, T* __restrict__ gw, int n, int C) {
    __shared__ float s[32][33];
    const int col = threadIdx.x & 31, grp = threadIdx.x >> 5, c = blockIdx.x * 32 + col;
    float v = 0.f;
    if (c < C) {
        int k = grp;
        for (; k + 7 * 32 < n; k += 8 * 32) {       // eight loads at a time
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = part[(long long)(k + 32 * j) * C + c];
#pragma unroll
            for (int j = 0; j < 8; ++j) v += x[j];
        }
        for (; k < n; k += 32) v += part[(long long)k * C + c];
    }
    s[grp][col] = v;
    __syncthreads();
    if (grp == 0 && c < C) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) t += s[k][col];
        st1(gw + c, t);
    }
}

// lanes per row and chunks per lane of a row of C elements.  A wave per row up to 1024 columns, a workgroup per row above: with a wave,
// 4096 columns of bf16 took 111 us forward and 180 us backward (16411 rows: 4.85 and 2.99 TB/s), with a workgroup 99 and 91 us (5.44 and
// 5.93 TB/s); at 1024 columns both read 5.4 TB/s and the wave needs no barrier.
struct RowShape {
    int lpr, cpl;
};
RowShape row_shape(int C) {
    const int chunks = C / 8;
    if (chunks <= 64) {
        int l = 8;
        while (l < chunks) l *= 2;
        return {l, 1};
    }
    if (chunks <= 128) return {64, (chunks + 63) / 64};
    return {256, (chunks + 255) / 256};
}
// workgroups of the backward: its partial sums of the weight gradient are read back by one more launch
int norm_bwd_blocks(long long M, int C) {
    const int rpb = 256 / row_shape(C).lpr;
    const long long b = (M + rpb - 1) / rpb;
    return (int)(b < 1024 ? b : 1024);
}

#define NORM_SHAPES(CASE) \
    CASE(8, 1) CASE(16, 1) CASE(32, 1) CASE(64, 1) CASE(64, 2) \
    CASE(256, 1) CASE(256, 2) CASE(256, 3) CASE(256, 4) CASE(256, 5) CASE(256, 6) CASE(256, 7) CASE(256, 8)

template <typename T>
int launch_norm_fwd(const NormFwd& a, int q8, hipStream_t st) {
    const RowShape s = row_shape(a.C);
    const long long b = (a.M + 256 / s.lpr - 1) / (256 / s.lpr);
    const dim3 grid((unsigned)(b < 4096 ? b : 4096));
#define CASE(L, N)                                                                                                   \
    if (s.lpr == L && s.cpl == N) {                                                                                  \
        if (q8 == 0) hipLaunchKernelGGL((k_rms_fwd<T, L, N, 0>), grid, dim3(256), 0, st, a);                         \
        else if (q8 == 1) hipLaunchKernelGGL((k_rms_fwd<T, L, N, 1>), grid, dim3(256), 0, st, a);                    \
        else hipLaunchKernelGGL((k_rms_fwd<T, L, N, 2>), grid, dim3(256), 0, st, a);                                 \
        return launched("sam3_seq_rms_norm_fwd");                                                                    \
    }
    NORM_SHAPES(CASE)
#undef CASE
    return sam3_seq_fail(ENOTSUP_, "rms norm: no kernel for %d columns", a.C);
}
template <typename T>
int launch_norm_bwd(const NormBwd& a, void* gw, hipStream_t st) {
    const RowShape s = row_shape(a.C);
    const int blocks = norm_bwd_blocks(a.M, a.C);
    bool found = false;
#define CASE(L, N)                                                                                                   \
    if (s.lpr == L && s.cpl == N) {                                                                                  \
        hipLaunchKernelGGL((k_rms_bwd<T, L, N>), dim3(blocks), dim3(256), 0, st, a);                                 \
        found = true;                                                                                                \
    }
    NORM_SHAPES(CASE)
#undef CASE
    if (!found) return sam3_seq_fail(ENOTSUP_, "rms norm: no kernel for %d columns", a.C);
    if (a.part) hipLaunchKernelGGL(k_rms_gw<T>, dim3((a.C + 31) / 32), dim3(1024), 0, st, (const float*)a.part, (T*)gw, blocks, a.C);
    return launched("sam3_seq_rms_norm_bwd");
}

int norm_check(int64_t M, int C, int dtype) {
    if (dtype != 0 && dtype != 1) return sam3_seq_fail(EINVAL_, "dtype must be 0 (bf16) or 1 (fp32), got %d", dtype);
    if (M < 0 || C <= 0 || C % 8) return sam3_seq_fail(EINVAL_, "rms norm: bad sizes [%lld, %d] (columns in multiples of 8)", (long long)M, C);
    if (C > 16384) return sam3_seq_fail(ENOTSUP_, "rms norm: at most 16384 columns, got %d", C);
    return 0;
}
bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }
// row pitches that keep 16-byte accesses aligned
bool bad_pitch(int64_t ld, int dtype) { return (ld % (dtype == 0 ? 8 : 4)) != 0; }

// ------------------------------------------------------------------------------------------------- rotary positions
// A workgroup takes TT tokens: their angles (one per token and pair, shared by all heads of q and k) are reduced in 64 bits to a
// fraction of a turn and put into LDS as (cos, sin); then the threads walk the tokens' chunks of 16 bytes (bf16), q's heads and k's in one
// row.  A rate is off by 2^-52 of itself or so, and with it the turns by 2^-54 of the position: 2^-24 of a turn, what fp32 holds of the
// fraction, up to positions of 2^30, and in proportion more behind them (2^-14 at 2^40).
struct RopeTable {
    double turns[128];
    unsigned char axis[128];
};
struct Rope {
    const void *q, *k, *pos;
    void *qo, *ko;
    long long q_st, q_sh, k_st, k_sh, pos_sa, pos_st, T;
    int Hq, Hk, D, pairs, TT;
    unsigned items, row_items, head_items;      // per workgroup, per token, per head
    unsigned mul_row, mul_head;                 // ceil(2^32 / row_items), ceil(2^32 / head_items)
    float sign;
};

__device__ __forceinline__ double position(const void* p, long long i, int type) {
    return type == 0 ? (double)((const int*)p)[i] : type == 1 ? (double)((const long long*)p)[i] : (double)((const float*)p)[i];
}

// 16 bytes from an address that is only aligned to an element
template <typename T>
__device__ __forceinline__ Raw8<T> load_any(const T* p) {
    Raw8<T> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}

// FORM 0: adjacent pairs; 1: halves, pairs % 8 == 0: a thread has 8 pairs; 2: halves, any number: a thread has 8 elements and reads their
// partners, which are not aligned (and which its neighbours read as their own: they come from the cache).
// 340 MB of bf16 (41472 tokens, 16 + 16 heads of 64, adjacent) in 69 us = 4.9 TB/s; halves 5.0 (heads of 128); halves of 13 pairs 3.1, the
// chunks across a middle or an end being read by elements.  Loading 2 to 4 chunks per thread before turning the first gained nothing.
template <typename T, int FORM>
__global__ __launch_bounds__(256) void k_rotary(Rope a, RopeTable tab, int pos_type) {
    extern __shared__ float2 cs[];      // [TT, pairs]
    const long long t0 = (long long)blockIdx.x * a.TT;
    const int nt = (int)(a.T - t0 < a.TT ? a.T - t0 : a.TT);
    for (int i = threadIdx.x; i < nt * a.pairs; i += 256) {
        const int t = i / a.pairs, p = i - t * a.pairs;
        const double turn = position(a.pos, tab.axis[p] * a.pos_sa + (t0 + t) * a.pos_st, pos_type) * tab.turns[p];
        float s, c;
        sincospif((float)(2.0 * (turn - rint(turn))), &s, &c);
        cs[i] = make_float2(c, s * a.sign);
    }
    __syncthreads();
    const unsigned total = (unsigned)nt * a.row_items;
    for (unsigned it = threadIdx.x; it < total; it += 256) {
        const unsigned t = a.row_items > 1 ? (unsigned)(((unsigned long long)it * a.mul_row) >> 32) : it;
        const unsigned rem = it - t * a.row_items;
        const unsigned head = a.head_items > 1 ? (unsigned)(((unsigned long long)rem * a.mul_head) >> 32) : rem;
        const bool isq = head < (unsigned)a.Hq;
        const int hd = isq ? head : head - a.Hq, d0 = (int)(rem - head * a.head_items) * 8;
        const long long row = t0 + t;
        const T* src = isq ? (const T*)a.q + row * a.q_st + hd * a.q_sh : (const T*)a.k + row * a.k_st + hd * a.k_sh;
        T* dst = isq ? (T*)a.qo + (row * a.Hq + hd) * a.D : (T*)a.ko + (row * a.Hk + hd) * a.D;
        const float2* c = cs + t * a.pairs;
        Raw8<T> v, w;
        float f[8], g[8];
        if (FORM == 0) {
            v.load(src + d0);
            v.get(f);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int p = d0 / 2 + j;
                if (p < a.pairs) {
                    const float x = f[2 * j], y = f[2 * j + 1];
                    f[2 * j] = x * c[p].x - y * c[p].y;
                    f[2 * j + 1] = x * c[p].y + y * c[p].x;
                }
            }
            v.set(f);
            v.store(dst + d0);
        } else if (FORM == 1) {
            const int d1 = d0 + a.pairs;
            if (d0 < a.pairs) {
                v.load(src + d0);
                w.load(src + d1);
                v.get(f);
                w.get(g);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 z = c[d0 + j];
                    const float x = f[j], y = g[j];
                    f[j] = x * z.x - y * z.y;
                    g[j] = x * z.y + y * z.x;
                }
                v.set(f);
                v.store(dst + d0);
                w.set(g);
                w.store(dst + d1);
            } else {
                v.load(src + d1);
                v.store(dst + d1);
            }
        } else {
            v.load(src + d0);
            if (d0 < 2 * a.pairs) {
                if (d0 + 8 <= a.pairs) {
                    w = load_any(src + d0 + a.pairs);
                } else if (d0 >= a.pairs && d0 + 8 <= 2 * a.pairs) {
                    w = load_any(src + d0 - a.pairs);
                } else {            // the chunks across the middle and the end
                    T e[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int i = d0 + j;
                        e[j] = src[i < a.pairs ? i + a.pairs : i < 2 * a.pairs ? i - a.pairs : i];
                    }
                    __builtin_memcpy(&w, e, sizeof(e));
                }
                v.get(f);
                w.get(g);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int i = d0 + j;
                    const bool second = i >= a.pairs;
                    const float2 z = c[i < 2 * a.pairs ? (second ? i - a.pairs : i) : 0];
                    const float r = second ? g[j] * z.y + f[j] * z.x : f[j] * z.x - g[j] * z.y;
                    if (i < 2 * a.pairs) f[j] = r;
                }
                v.set(f);
            }
            v.store(dst + d0);
        }
    }
}

constexpr long long MOST_BLOCKS = (1ll << 32) / 256 - 1;
unsigned magic(unsigned d) { return (unsigned)((0x100000000ull + d - 1) / d); }

}  // namespace

extern "C" {

const char* sam3_seq_last_error(void) { return g_err; }

int sam3_seq_rms_norm_fwd(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, void* y, void* h_out,
                          void* h_low, float* rstd_out, void* q8, float* scales, int group, int fmt, int64_t M, int C, float eps, int dtype,
                          void* stream) {
    sam3_seq_clear_error();
    if (int rc = norm_check(M, C, dtype)) return rc;
    if (!(eps >= 0.f) || eps > 3.0e38f) return sam3_seq_fail(EINVAL_, "rms norm: eps must be finite and not negative");
    if (h_low && (dtype != 0 || !h_out)) return sam3_seq_fail(EINVAL_, "rms norm: h_low goes with a bf16 h_out");
    if ((q8 == nullptr) != (scales == nullptr)) return sam3_seq_fail(EINVAL_, "rms norm: the 8-bit output needs its scales");
    if (q8 && fmt != SAM3_FP8_E4M3 && fmt != SAM3_FP8_E5M2) return sam3_seq_fail(EINVAL_, "rms norm: unknown 8-bit format %d", fmt);
    if (q8 && group && ((group != 32 && group != 64 && group != 128) || C % group))
        return sam3_seq_fail(EINVAL_, "rms norm: scale groups are 32, 64 or 128 columns that divide %d, got %d", C, group);
    if (M == 0) return 0;
    if (!x || !weight || (!y && !q8)) return sam3_seq_fail(EINVAL_, "rms norm: null pointer");
    if (misaligned(x) || misaligned(residual) || misaligned(weight) || misaligned(y) || misaligned(h_out) || ((uintptr_t)q8 & 7) || ((uintptr_t)h_low & 1))
        return sam3_seq_fail(EINVAL_, "rms norm: tensors must be 16-byte aligned");
    if (ldx < C || bad_pitch(ldx, dtype) || (residual && (ldr < C || bad_pitch(ldr, dtype))))
        return sam3_seq_fail(EINVAL_, "rms norm: bad row pitch");
    const NormFwd a{x, residual, weight, y, h_out, (unsigned short*)h_low, rstd_out, (unsigned char*)q8, scales, ldx, ldr, M, C, !group ? 0 : group == 32 ? 5 : group == 64 ? 6 : 7, eps,
                    fmt == SAM3_FP8_E4M3 ? 448.f : 57344.f};
    const int q = !q8 ? 0 : fmt == SAM3_FP8_E4M3 ? 1 : 2;
    return dtype == 0 ? launch_norm_fwd<bf16_t>(a, q, (hipStream_t)stream) : launch_norm_fwd<float>(a, q, (hipStream_t)stream);
}

size_t sam3_seq_rms_norm_bwd_workspace_bytes(int64_t M, int C) {
    return M > 0 && C > 0 && C % 8 == 0 && C <= 16384 ? (size_t)norm_bwd_blocks(M, C) * C * sizeof(float) : 0;
}

int sam3_seq_rms_norm_bwd(const void* gy, const void* gh, const void* h, int64_t ldh, const void* h_low, const void* weight, const float* rstd, void* gx,
                          void* gw, int64_t M, int C, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    sam3_seq_clear_error();
    if (int rc = norm_check(M, C, dtype)) return rc;
    if (M == 0) return gw ? sam3_seq_fail(EINVAL_, "rms norm: no rows to sum a weight gradient over") : 0;
    if (!gy || !h || !weight || !rstd || (!gx && !gw)) return sam3_seq_fail(EINVAL_, "rms norm: null pointer");
    if (misaligned(gy) || misaligned(gh) || misaligned(h) || misaligned(weight) || misaligned(gx))
        return sam3_seq_fail(EINVAL_, "rms norm: tensors must be 16-byte aligned");
    if (h_low && (dtype != 0 || ldh != C || ((uintptr_t)h_low & 1))) return sam3_seq_fail(EINVAL_, "rms norm: h_low goes with a contiguous bf16 h");
    if (ldh < C || bad_pitch(ldh, dtype)) return sam3_seq_fail(EINVAL_, "rms norm: bad row pitch");
    if (gw && (!workspace || workspace_bytes < sam3_seq_rms_norm_bwd_workspace_bytes(M, C)))
        return sam3_seq_fail(ENOMEM_, "rms norm: workspace too small: %zu < %zu", workspace_bytes, sam3_seq_rms_norm_bwd_workspace_bytes(M, C));
    const NormBwd a{gy, gh, h, weight, (const unsigned short*)h_low, rstd, gx, gw ? (float*)workspace : nullptr, ldh, M, C};
    return dtype == 0 ? launch_norm_bwd<bf16_t>(a, gw, (hipStream_t)stream) : launch_norm_bwd<float>(a, gw, (hipStream_t)stream);
}

int sam3_seq_rotary(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, void* q_out, void* k_out,
                    const void* positions, int64_t pos_sa, int64_t pos_st, int pos_type, int axes, const double* turns,
                    const unsigned char* axis, int pairs, int halves, int inverse, int64_t T, int Hq, int Hk, int D, int dtype,
                    void* stream) {
    sam3_seq_clear_error();
    if (dtype != 0 && dtype != 1) return sam3_seq_fail(EINVAL_, "dtype must be 0 (bf16) or 1 (fp32), got %d", dtype);
    if (!k) Hk = 0;
    if (T < 0 || Hq <= 0 || Hk < 0 || D <= 0 || D % 8 || D > 256) return sam3_seq_fail(EINVAL_, "rotary: bad sizes (head size in multiples of 8, at most 256)");
    if (Hq > 1024 || Hk > 1024) return sam3_seq_fail(ENOTSUP_, "rotary: at most 1024 heads");
    if (pairs <= 0 || 2 * pairs > D || !turns || !axis) return sam3_seq_fail(EINVAL_, "rotary: %d pairs do not fit a head of %d", pairs, D);
    if (pos_type < 0 || pos_type > 2 || axes <= 0) return sam3_seq_fail(EINVAL_, "rotary: bad positions");
    RopeTable tab = {};
    for (int i = 0; i < pairs; ++i) {
        if (axis[i] >= axes) return sam3_seq_fail(EINVAL_, "rotary: pair %d wants axis %d of %d", i, (int)axis[i], axes);
        tab.turns[i] = turns[i];
        tab.axis[i] = axis[i];
    }
    if (T == 0) return 0;
    if (!q || !q_out || !positions || (k && !k_out)) return sam3_seq_fail(EINVAL_, "rotary: null pointer");
    if (misaligned(q) || misaligned(k) || misaligned(q_out) || misaligned(k_out) || bad_pitch(q_st, dtype) || bad_pitch(q_sh, dtype) ||
        (k && (bad_pitch(k_st, dtype) || bad_pitch(k_sh, dtype))))
        return sam3_seq_fail(EINVAL_, "rotary: tensors and strides must keep 16-byte accesses aligned");
    const int form = !halves ? 0 : pairs % 8 == 0 ? 1 : 2;
    const int per_head = form == 1 ? (D - pairs) / 8 : D / 8;
    Rope a{q, k, positions, q_out, k_out, q_st, q_sh, k_st, k_sh, pos_sa, pos_st, T, Hq, Hk, D, pairs, 0, 0, 0, 0, 0, 0, inverse ? -1.f : 1.f};
    a.head_items = per_head;
    a.row_items = (unsigned)per_head * (Hq + Hk);
    a.TT = T >= 16384 ? 8 : T >= 2048 ? (int)(T / 2048) : 1;      // tokens that share a table, as long as there are 2048 workgroups
    a.mul_head = magic(a.head_items);
    a.mul_row = magic(a.row_items);
    if ((uint64_t)a.TT * a.row_items * a.row_items >= 0x100000000ull) a.TT = 1;
    if ((uint64_t)a.row_items * a.row_items >= 0x100000000ull) return sam3_seq_fail(ENOTSUP_, "rotary: too many elements in a token's heads");
    // (a grid has fewer than 2^32 threads: from 2^27 tokens on, more of them share a table)
    if ((T + a.TT - 1) / a.TT > MOST_BLOCKS) a.TT = (int)(T / MOST_BLOCKS + 1 < 1024 ? T / MOST_BLOCKS + 1 : 1024);
    const long long blocks = (T + a.TT - 1) / a.TT;
    if (blocks > MOST_BLOCKS || (uint64_t)a.TT * a.row_items * a.row_items >= 0x100000000ull || (int64_t)a.TT * pairs > 8192)
        return sam3_seq_fail(ENOTSUP_, "rotary: too many tokens");
    const size_t lds = (size_t)a.TT * pairs * sizeof(float2);
    hipStream_t st = (hipStream_t)stream;
#define ROT(TY, F) hipLaunchKernelGGL((k_rotary<TY, F>), dim3((unsigned)blocks), dim3(256), lds, st, a, tab, pos_type)
    if (dtype == 0) { if (form == 0) ROT(bf16_t, 0); else if (form == 1) ROT(bf16_t, 1); else ROT(bf16_t, 2); }
    else { if (form == 0) ROT(float, 0); else if (form == 1) ROT(float, 1); else ROT(float, 2); }
#undef ROT
    return launched("sam3_seq_rotary");
}

}  // extern "C"
