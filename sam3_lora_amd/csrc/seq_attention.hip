// sam3_lora_amd -- attention over packed sequences with grouped heads (gfx950): C-ABI of include/sam3_seq_amd.h.
//
//   o_i = sum_j p_ij v_j,   p_ij = exp(c q_i k_j - lse_i)    over the keys j that query i sees
//   D_i = go_i o_i,  dS_ij = p_ij (go_i v_j - D_i),  gq_i = c sum_j dS_ij k_j,  gk_j = c sum_i dS_ij q_i,  gv_j = sum_i p_ij go_i
//
// The heads that share a key head are rows of one matrix: row r of (sequence, key head) is token r / G, head r % G of the group, so
// one tile of keys serves the whole group, and the sums over the group in gk and gv are the sums over the rows.
//
// Every product is a 32 x 32 x 16 matrix instruction whose result has one row (forward, gq) or one key (gk, gv) per lane, and 16 of
// the other index in registers: statistics of a row are a lane's own scalars, and the result turns into the second operand of the
// next product without leaving the lane -- the sum over k runs in the order the registers hold it, and the other operand, read
// from LDS by transposing reads, follows that order.
//
// Prompts are bound by the order inside a wave: scores, maximum, exponentials and the second product follow each other, and the two or three
// waves of a SIMD do not cover the waits.  By counters (with 32 / 8 heads of 128 and 8192 tokens that all see each other; heads of 64: 16, 4 x 5184
// tokens) the matrix cores are busy 47, 61 and 52 % of the cycles in the forward, gq and gk, gv (64: 38, 47 and 47 %), vector units 7 to 17 %,
// LDS 20 to 39 % without bank conflicts, at 1.6 to 1.9 GHz of 2.4: no unit is full.  The forward runs at 1000 TF, gq at 1160 (three products) and
// gk, gv at 1155 (four), where a library product of 8192^3 runs at 1295; heads of 64 at 825, 965 and 1000.  The backward recomputes the
// scores in both of its kernels, seven products for the five of the formulas: one pass with sums in memory would need atomics, whose order
// changes the result, or a second pass over 32-bit partial sums.
#include "seq_common.inc"

#include <type_traits>

#include "sam3_seq_amd.h"

using namespace seq;

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Attn {
    const void *q, *k, *v, *go, *o;
    void *out, *gq, *gk, *gv;
    float *lse;                 // [Tq, Hq]
    float *rowstat;             // [3, Hk, Tq, G] of the backward: exponent base (16 bits: with the sum's logarithm), D, 1 / sum (32 bits only)
    float2* stats;              // [Tq, Hq]: exponent base (powers of two) and 1 / sum of each row; 0 for a row that sees no key
    const int *cu_q, *cu_k, *len_k;
    long long q_st, q_sh, k_st, k_sh, v_st, v_sh, go_st, go_sh;
    long long Tq, Tk;
    int B, Hq, Hk, G, D, causal;
    float scale;
};

// operand of a 32 x 32 x 16 product: lane l holds row (or column) l % 32, and 8 of the 16 k
template <typename T> struct Frag;
template <> struct Frag<bf16_t> { bf16x8 v; };
template <> struct Frag<float> { float v[8]; };

__device__ __forceinline__ f32x16 mma(const Frag<bf16_t>& a, const Frag<bf16_t>& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
// 32 bits: eight instructions of two k each; instruction j takes element j of both lane halves, of A and B alike
__device__ __forceinline__ f32x16 mma(const Frag<float>& a, const Frag<float>& b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}
// index along the result's register side: register i of lane half h
__device__ __forceinline__ int reg_row(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }

// eight elements of one row from global memory (zeros where `on` is false)
__device__ __forceinline__ Frag<bf16_t> frag_global(const bf16_t* p, bool on) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (on) u = *reinterpret_cast<const uint4*>(p);
    return Frag<bf16_t>{__builtin_bit_cast(bf16x8, u)};
}
__device__ __forceinline__ Frag<float> frag_global(const float* p, bool on) {
    Frag<float> f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (on) {
        a = *reinterpret_cast<const float4*>(p);
        b = *reinterpret_cast<const float4*>(p + 4);
    }
    f.v[0] = a.x; f.v[1] = a.y; f.v[2] = a.z; f.v[3] = a.w;
    f.v[4] = b.x; f.v[5] = b.y; f.v[6] = b.z; f.v[7] = b.w;
    return f;
}
// registers 8 t .. 8 t + 7 of a result as the k-step t of the next product's second operand
__device__ __forceinline__ void frag_of(Frag<bf16_t>& f, const float* p) {
    f.v = __builtin_bit_cast(bf16x8, make_uint4(pack2(p[0], p[1]), pack2(p[2], p[3]), pack2(p[4], p[5]), pack2(p[6], p[7])));
}
__device__ __forceinline__ void frag_of(Frag<float>& f, const float* p) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = p[j];
}

// What that rounding to 16 bits took away, as one more operand.  Weights and dS rounded once leave a result sqrt(2) of its own rounding's error,
// more where a few of them decide it, and in gq, whose keys are weighted most where they lie along q, up to 1.57 for heads of 32 (4 x 2000
// to 32 x 500 tokens; 1.5 for 64, 1.47 for 128).  The products with the rest are taken (FINE; the error is 1.0 to 1.1 then) where they are
// cheap or needed most: one tile of rows in the forward (decode of 24 requests 417 -> 423 us; with more tiles, 64 new tokens over 32768 keys,
// 134 -> 148), gq in tiles of 32 (120 -> 128 at 4 x 128 tokens over 4096 keys) and for heads up to 32 (4 x 4096 tokens 177 -> 224; for heads
// of 64 it would be 715 -> 906), gk and gv of one wave (text prompts 12.4 -> 12.5; with four waves it would be 480 -> 600 at 4096 tokens).
__device__ __forceinline__ void rest_of(Frag<bf16_t>& f, const Frag<bf16_t>& hi, const float* p) {
    float r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = p[j] - (float)hi.v[j];
    frag_of(f, r);
}
__device__ __forceinline__ void rest_of(Frag<float>&, const Frag<float>&, const float*) {}

// A tile of rows in LDS: rows of DP elements in chunks of 16 bytes, the chunks of a row permuted by an exclusive or with f(row).  LDS has
// 64 banks of 4 bytes, a line of 16 chunks.  Reading rows, 16 lanes read the same chunk of 16 neighbouring rows: f takes them to 16
// different places of a line.  Reading columns, lanes read the same four chunks of 4 neighbouring rows: f's upper bits come from the
// row's lower ones, so that these fill a line too.  (With f = row % 8 two thirds of the LDS's busy time were bank conflicts.)
template <typename T, int DP>
struct Tile {
    static constexpr int EPC = 16 / sizeof(T);          // elements per chunk
    static constexpr int CPR = DP / EPC;                // chunks per row
    static constexpr int ROWB = DP * sizeof(T);
    static constexpr int PERIOD = 16;                   // f(row) = f(row + 16)
    static __device__ __forceinline__ int f(int row) {
        if (CPR >= 16) return ((row & 3) << 2) | ((row >> 2) & 3);
        if (CPR == 8) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
        return (row >> 2) & 3;
    }
    static __device__ __forceinline__ int chunk_at(int row, int c) { return row * ROWB + ((c ^ f(row)) << 4); }
    // k-step s (16 elements) of row `row`: elements 16 s + 8 h .. + 7
    static __device__ __forceinline__ Frag<T> row_frag(const char* t, int row, int s, int h) {
        Frag<T> r;
        if constexpr (sizeof(T) == 2) {
            r.v = *reinterpret_cast<const bf16x8*>(t + chunk_at(row, 2 * s + h));
        } else {
            const float4 a = *reinterpret_cast<const float4*>(t + chunk_at(row, 4 * s + 2 * h));
            const float4 b = *reinterpret_cast<const float4*>(t + chunk_at(row, 4 * s + 2 * h + 1));
            r.v[0] = a.x; r.v[1] = a.y; r.v[2] = a.z; r.v[3] = a.w;
            r.v[4] = b.x; r.v[5] = b.y; r.v[6] = b.z; r.v[7] = b.w;
        }
        return r;
    }
    // the tile's transpose: lane l = column 32 dt + l % 32, k = rows row0 + reg_row order: {0..3} + 4 h and 8 + {0..3} + 4 h
    static __device__ __forceinline__ Frag<T> col_frag(const char* t, int row0, int dt, int lane) {
        Frag<T> r;
        const int h = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            // 16 lanes read a 4 x 16 block and get its columns: lane i addresses row i / 4, elements 4 (i % 4) .. + 3
            const int i = lane & 15, c = dt * 4 + ((lane >> 4) & 1) * 2 + ((i & 3) >> 1), off = (i & 1) * 8;
            const int ra = row0 + 4 * h + (i >> 2), rb = ra + 8;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(t + chunk_at(ra, c) + off));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(t + chunk_at(rb, c) + off));
            const s16x8 both = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            r.v = __builtin_bit_cast(bf16x8, both);
        } else {
            const int d = dt * 32 + (lane & 31);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                r.v[j] = *reinterpret_cast<const float*>(t + chunk_at(row0 + 4 * h + (j & 3) + 8 * (j >> 2), d >> 2) + (d & 3) * 4);
        }
        return r;
    }
};

// where a sequence lies; begin / count clamped to the tensors
struct Span {
    long long begin;
    int n;
};
__device__ __forceinline__ Span span(const int* cu, const int* len, int b, long long total) {
    long long s = cu[b], e = len ? s + len[b] : cu[b + 1];
    s = s < 0 ? 0 : s > total ? total : s;
    e = e < s ? s : e > total ? total : e;
    return Span{s, (int)(e - s)};
}
// rows of no sequence: [0, cu[0]) and [cu[B], total)
struct Rest {
    long long head, tail, n;
    __device__ __forceinline__ long long row(long long i) const { return i < head ? i : tail + (i - head); }
};
__device__ __forceinline__ Rest rest(const int* cu, int B, long long total) {
    long long s = cu[0], e = cu[B];
    s = s < 0 ? 0 : s > total ? total : s;
    e = e < s ? s : e > total ? total : e;
    return Rest{s, e, s + (total - e)};
}
__device__ __forceinline__ int seen_keys(int token, int nq, int nk, int causal) {
    if (!causal) return nk;
    const long long j = (long long)token + 1 + nk - nq;
    return j < 0 ? 0 : j > nk ? nk : (int)j;
}

// 1 / sum of a row's weights.  There are none where the row sees no key (zeros come out), and where all its scores are -inf (0 / 0)
__device__ __forceinline__ float one_over(float sum, int keys) { return sum != 0.f ? 1.f / sum : keys > 0 ? NAN : 0.f; }

// rows of one (sequence, head group) as addresses: row r -> token r / G, head kv * G + r % G
struct Rows {
    long long begin, st, sh;
    int G, head0;
    __device__ __forceinline__ long long at(int r) const {
        const int t = r / G;
        return (begin + t) * st + (long long)(head0 + (r - t * G)) * sh;
    }
};

// ROWS rows (n of them there, the others zeros) of DP elements (D of them there) into LDS by NT threads.
// CHECK: infinities and NaN become zeros, and the answer says whether there were any.  A product over a tile that some of its rows
// only see a part of multiplies what they do not see by zero, which a non-finite element would turn into NaN; such tiles are
// staged with the check, and the rows that do see such an element get its effect afterwards (spoils(), add_nonfinite(), add_to_row()).
__device__ __forceinline__ bool finite_bits(unsigned u, bf16_t) { return (u & 0x7f80u) != 0x7f80u && (u & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ bool finite_bits(unsigned u, float) { return (u & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ unsigned only_finite(unsigned u, bf16_t) {
    return ((u & 0x7f80u) == 0x7f80u ? 0u : u & 0xffffu) | ((u & 0x7f800000u) == 0x7f800000u ? 0u : u & 0xffff0000u);
}
__device__ __forceinline__ unsigned only_finite(unsigned u, float) { return (u & 0x7f800000u) == 0x7f800000u ? 0u : u; }

template <typename T, int DP, int ROWS, bool CHECK, int NT = 256, typename ADDR>
__device__ __forceinline__ bool stage(char* lds, const T* base, int n, int D, ADDR addr) {
    typedef Tile<T, DP> L;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < (ROWS * L::CPR + NT - 1) / NT; ++i) {
        const int p = i * NT + threadIdx.x % NT, row = p / L::CPR, c = p % L::CPR;
        if (ROWS * L::CPR % NT && row >= ROWS) break;
        uint4 u = make_uint4(0, 0, 0, 0);
        if (row < n && c * L::EPC < D) u = *reinterpret_cast<const uint4*>(base + addr(row) + c * L::EPC);
        if (CHECK && !(finite_bits(u.x, T()) && finite_bits(u.y, T()) && finite_bits(u.z, T()) && finite_bits(u.w, T()))) {
            bad = true;
            u = make_uint4(only_finite(u.x, T()), only_finite(u.y, T()), only_finite(u.z, T()), only_finite(u.w, T()));
        }
        *reinterpret_cast<uint4*>(lds + L::chunk_at(row, c)) = u;
    }
    return bad;
}
// does a row hold an infinity or a NaN (rare path, as what follows: the rows are read 8 elements at a time, and no further than it takes)
template <typename T>
__device__ bool spoils(const T* row, int D) {
#pragma unroll 1
    for (int d = 0; d < D; d += 8) {
        Raw8<T> x;
        float f[8], s = 0.f;
        x.load(row + d);
        x.get(f);
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(f[j], 0.f, s);
        if (s != 0.f) return true;
    }
    return false;
}
template <typename T>
__device__ float dot(const T* a, const T* b, int D) {
    float s = 0.f;
#pragma unroll 1
    for (int d = 0; d < D; d += 8) {
        Raw8<T> x, y;
        float f[8], g[8];
        x.load(a + d);
        y.load(b + d);
        x.get(f);
        y.get(g);
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(f[j], g[j], s);
    }
    return s;
}
// out += w x in memory, by a lane half's columns (store_cols()); rest: only where that is not finite, since the finite part is in it already.
// Whether all of the columns are NaN now: nothing that is added later changes them.
template <typename T>
__device__ bool add_to_row(T* out, float w, const T* x, int D, int h, bool rest) {
    bool nan = true;
#pragma unroll 1
    for (int d = 4 * h; d < D; d += 8)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float y = w * ld1(x + d + j), z = ld1(out + d + j), sum = rest && fabsf(y) <= 3.402823466e38f ? z : z + y;
            nan &= sum != sum;
            st1(out + d + j, sum);
        }
    return nan;
}
// Clears the rows of a staged tile that hold an infinity or a NaN: their products with the others of the tile come to nothing then.
template <typename T, int DP, int NT>
__device__ void clear_spoilt(char* lds, const T* base, long long st, int n, int D) {
    for (int row = threadIdx.x % NT; row < n; row += NT)
        if (spoils(base + row * st, D))
            for (int c = 0; c < Tile<T, DP>::ROWB; c += 16) *reinterpret_cast<uint4*>(lds + row * Tile<T, DP>::ROWB + c) = make_uint4(0, 0, 0, 0);
}

// the result's registers of one 32-column block of a row, four neighbours at a time
template <typename T>
__device__ __forceinline__ void store_cols(T* row, const f32x16& acc, int dt, int h, int D, float mul) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int d = dt * 32 + 8 * g + 4 * h;
        if (d < D) {
            const float a = acc[4 * g] * mul, b = acc[4 * g + 1] * mul, c = acc[4 * g + 2] * mul, e = acc[4 * g + 3] * mul;
            if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(row + d) = make_uint2(pack2(a, b), pack2(c, e));
            else *reinterpret_cast<float4*>(row + d) = make_float4(a, b, c, e);
        }
    }
}
template <typename T>
__device__ __forceinline__ void zero_row(T* row, int D, int lane, int lanes) {
    for (int d = lane * 8; d < D; d += lanes * 8) {
        Raw8<T> z;
        const float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        z.set(f);
        z.store(row + d);
    }
}

// the infinities and NaN of n value rows into the results of a row that sees them: whatever their weight, they decide it
template <typename T, int DT>
__device__ __forceinline__ void add_nonfinite(f32x16* acc, const T* v, long long st, int n, int D, int h) {
    for (int j = 0; j < n; ++j)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int e = d * 32 + reg_row(i, h);
                const float x = e < D ? ld1(v + j * st + e) : 0.f;
                if (!(fabsf(x) <= 3.402823466e38f)) acc[d][i] += x;
            }
}

constexpr int BM = 128;      // rows of a workgroup: 4 waves of 32

// Which (sequence, key head) and which of its tiles a workgroup takes.  Workgroups go round the 8 XCDs in turn, and each XCD has its own
// L2: the tiles of one pair, which read the same keys, stay on one XCD where the number of pairs is a multiple of 8, and on 2, 4 or 8
// of them otherwise, so that all are busy.  The last tiles of a causal sequence have the most keys and go first.
struct Place {
    int pair, tile;
};
__host__ __device__ inline int xcds_per_pair(int pairs) { return pairs % 8 == 0 ? 1 : pairs % 4 == 0 ? 2 : pairs % 2 == 0 ? 4 : 8; }
__host__ __device__ inline long long places(int pairs, int tiles) {
    const int s = xcds_per_pair(pairs);
    return (long long)pairs * ((tiles + s - 1) / s) * s;
}
__device__ __forceinline__ Place place(unsigned id, int pairs, int tiles) {
    const int s = xcds_per_pair(pairs), lanes = 8 / s, per = (tiles + s - 1) / s;
    const int xcd = id & 7, slot = id >> 3;
    const int tile = (slot % per) * s + xcd / lanes;
    return Place{xcd % lanes + lanes * (slot / per), tiles - 1 - tile};        // tile < 0: none
}
// The longest sequence's tiles for every pair are far too many where the others are much shorter, or where nobody said how long they are.
// Then the tiles are listed instead: sequence b, whose rows begin at row cu[b] * g of all, has the places from cu[b] * g / PER + b on, at
// least as many as it has tiles, and a workgroup finds its sequence among them, 64 at a time.  The heads of a place are neighbours.
__device__ __forceinline__ long long first_place(const int* cu, int b, int g, int per, long long total) {
    const long long c = cu[b];
    return (c < 0 ? 0 : c > total ? total : c) * g / per + b;
}
template <int PER>
__device__ __forceinline__ Place listed(unsigned id, const int* cu, int B, int Hk, int g, long long total) {
    const int lane = threadIdx.x & 63, kv = (int)(id % (unsigned)Hk);
    const long long slot = id / (unsigned)Hk;
    int lo = 0, n = B;              // the sequence is one of lo .. lo + n - 1
    while (n > 1) {
        const int apart = (n + 63) / 64, at = lane * apart;
        const int below = __popcll(__ballot(at < n && first_place(cu, lo + min(at, n - 1), g, PER, total) <= slot));
        const int skip = (below > 1 ? below - 1 : 0) * apart;
        lo += skip;
        n = min(apart, n - skip);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const long long tile = slot - first_place(cu, lo, g, PER, total);
    return Place{lo * Hk + kv, (int)(tile < 0 ? -1 : tile)};
}

// 16 bytes per lane straight into LDS, lane l's to lds + 16 l, from an address of the wave and 32 bits of the lane.  The instruction is
// written out because the compiler would wait for every such load before any later read of LDS, and the loads of the next tile have to
// stay in flight; whoever reads waits at the barrier in front (wait_loads).
// Its destination is M0; the address goes through a scalar move inside the block: a scalar register that a vector instruction wrote (the
// compiler's readfirstlane) may only be read by a memory instruction five wait states later, by a scalar one at once.
__device__ __forceinline__ unsigned lds_at(const void* lds) {
    return (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)lds);
}
__device__ __forceinline__ const void* of_wave(const void* p) {
    const unsigned long long u = (unsigned long long)p;
    const unsigned lo = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)u), hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(u >> 32));
    return (const void*)((unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ void load_to_lds(const void* base, unsigned off, unsigned lds) {
    unsigned long long tmp;
    asm volatile("s_mov_b32 m0, %1\n\ts_mov_b64 %0, %3\n\tglobal_load_lds_dwordx4 %2, %0"
                 : "=&s"(tmp) : "s"(lds), "v"(off), "s"(of_wave(base)) : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds(const void* p, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}
// 4 bytes per lane
// (The compiler warns that M0 in the clobbers is reserved.  Nothing else in these kernels uses it: the only M0 in their assembly is this.)
__device__ __forceinline__ void word_to_lds(const void* base, unsigned off, unsigned lds) {
    unsigned long long tmp;
    asm volatile("s_mov_b32 m0, %1\n\ts_mov_b64 %0, %3\n\tglobal_load_lds_dword %2, %0"
                 : "=&s"(tmp) : "s"(lds), "v"(off), "s"(of_wave(base)) : "memory", "m0");
}
// Waits until at most N loads are under way.  The builtin (the compiler then knows that its own earlier loads have arrived: it would
// otherwise wait for one of them inside the loop, and with it for the loads into LDS that it does not know of), and a fence for it.
template <int N>
__device__ __forceinline__ void wait_loads() {
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
    asm volatile("" ::: "memory");
}
// A tile of whole rows into LDS by NT threads without passing through registers, in rounds of RPI rows.  The chunks' permutation is on
// the address that a lane reads; chunks behind the head's end are left alone (they were cleared once).
template <typename T, int DP, int ROWS, int NT = 256>
struct Dma {
    typedef Tile<T, DP> L;
    static constexpr int RPI = NT / L::CPR, N = ROWS / RPI, P = RPI >= L::PERIOD ? 1 : L::PERIOD / RPI;
    static_assert(ROWS % RPI == 0, "whole rounds");
    unsigned off[P];        // bytes from the tile's first row, for the rounds i = p, p + P, ... (a tile spans less than 2^31: check_tensor)
    bool on[P];
    __device__ __forceinline__ Dma(long long st, int D) {
        const int row = (threadIdx.x % NT) / L::CPR, slot = threadIdx.x % L::CPR;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int e = (slot ^ L::f(p * RPI + row)) * L::EPC;
            off[p] = (unsigned)((row * st + e) * (long long)sizeof(T));
            on[p] = e < D;
        }
    }
    // lds: where the wave's first 1024 bytes go (the tile's address + 1024 times the wave)
    __device__ __forceinline__ void load(const T* tile, long long st, unsigned lds) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (on[i % P])
                load_to_lds(tile + i * RPI * st, off[i % P], lds + i * NT * 16);
    }
};

// ---------------------------------------------------------------------------------------------------------- forward
// One pass over the keys with a running maximum and sum per row.  The maximum in use only follows when a row's new one is 2^8 above
// it: weights stay below 2^8 (their relative precision does not change), and the accumulators are hardly ever rescaled.
template <typename T, int DP>
struct FwdCfg {
    static constexpr int BN = sizeof(T) * DP > 256 ? 32 : 64;       // keys of a step
};

template <typename T, int DP, int BN>
struct FwdState {
    typedef Tile<T, DP> L;
    static constexpr int KS = DP / 16, DT = DP / 32, SUBS = BN / 32;
    Frag<T> qf[KS];
    f32x16 acc[DT];
    float base, l;      // exponent base in powers of two, this half-wave's part of the sum

    template <bool MASK, bool FINE = false>
    __device__ __forceinline__ void step(const char* lk, const char* lv, int lane, float c2, int left) {
        const int h = lane >> 5;
        f32x16 s[SUBS];
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub) {
            s[sub] = zero16();
#pragma unroll
            for (int i = 0; i < KS; ++i) s[sub] = mma(L::row_frag(lk, sub * 32 + (lane & 31), i, h), qf[i], s[sub]);
        }
        float mx = -INFINITY;
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (MASK && sub * 32 + reg_row(i, h) >= left) s[sub][i] = -INFINITY;
                mx = fmaxf(mx, s[sub][i]);
            }
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * c2;
        if (__any(mx > base + 8.f)) {
            const float next = mx > base + 8.f ? mx : base, alpha = __builtin_amdgcn_exp2f(base - next);
            base = next;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[d][i] *= alpha;
        }
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub) {
            float p[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                p[i] = __builtin_amdgcn_exp2f(fmaf(s[sub][i], c2, -base));
                l += p[i];
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                Frag<T> pf, pr;
                frag_of(pf, p + 8 * t);
                if (FINE) rest_of(pr, pf, p + 8 * t);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const Frag<T> vf = L::col_frag(lv, sub * 32 + 16 * t, d, lane);
                    acc[d] = mma(vf, pf, acc[d]);
                    if (FINE && sizeof(T) == 2) acc[d] = mma(vf, pr, acc[d]);
                }
            }
        }
    }
};

// (three waves share a SIMD's registers up to heads of 128 bytes: 4 x 5184, heads of 64: 599 -> 545 us)
template <typename T, int DP, bool LISTED>
__global__ __launch_bounds__(256, (sizeof(T) * DP > 256 ? 1 : sizeof(T) * DP <= 128 ? 3 : 2)) void k_attn_fwd(Attn a, int tiles, unsigned first_rest) {
    typedef Tile<T, DP> L;
    constexpr int BN = FwdCfg<T, DP>::BN, TB = BN * L::ROWB;
    constexpr int KS = DP / 16, DT = DP / 32;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TB];        // two tiles of keys and values
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    T* out = (T*)a.out;
    if (blockIdx.x >= first_rest) {         // rows of no sequence
        const Rest z = rest(a.cu_q, a.B, a.Tq);
        for (long long i = (long long)(blockIdx.x - first_rest) * 32 + (threadIdx.x >> 3); i < z.n * a.Hq; i += (long long)(gridDim.x - first_rest) * 32) {
            const long long r = z.row(i / a.Hq) * a.Hq + i % a.Hq;
            zero_row(out + r * a.D, a.D, threadIdx.x & 7, 8);
            if (a.lse && (threadIdx.x & 7) == 0) a.lse[r] = -INFINITY;
        }
        return;
    }
    const Place pl = LISTED ? listed<BM>(blockIdx.x, a.cu_q, a.B, a.Hk, a.G, a.Tq) : place(blockIdx.x, a.B * a.Hk, tiles);
    if (pl.tile < 0) return;
    const int b = pl.pair / a.Hk, kv = pl.pair - b * a.Hk;
    const Span sq = span(a.cu_q, nullptr, b, a.Tq), sk = span(a.cu_k, a.len_k, b, a.Tk);
    const int R = sq.n * a.G;
    if ((long long)pl.tile * BM >= R) return;
    const Rows qrows{sq.begin, a.q_st, a.q_sh, a.G, kv * a.G};
    const T *k = (const T*)a.k + sk.begin * a.k_st + kv * a.k_sh, *v = (const T*)a.v + sk.begin * a.v_st + kv * a.v_sh;
    const float c2 = a.scale * LOG2E;
    const Dma<T, DP, BN> dk(a.k_st, a.D), dv(a.v_st, a.D);
    const unsigned at_lds = lds_at(lds) + wave * 1024;
    if (a.D < DP) {
        for (int i = threadIdx.x; i < 4 * TB / 16; i += 256) reinterpret_cast<uint4*>(lds)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    for (long long rr = (long long)pl.tile * BM; rr < R; rr += (long long)tiles * BM) {
        const int r0 = (int)rr;
        const int row = r0 + wave * 32 + (lane & 31);
        const bool live = row < R;
        const int jmax = live ? seen_keys(row / a.G, sq.n, sk.n, a.causal) : 0;
        const int last = min(r0 + BM, R) - 1;
        const int jend = seen_keys(last / a.G, sq.n, sk.n, a.causal);           // keys that any row of the tile sees
        const int jall = seen_keys(r0 / a.G, sq.n, sk.n, a.causal);             // keys that every row of the tile sees
        const int jwave = r0 + wave * 32 < R ? seen_keys(min(r0 + wave * 32 + 31, last) / a.G, sq.n, sk.n, a.causal) : 0;
        FwdState<T, DP, BN> st;
#pragma unroll
        for (int s = 0; s < KS; ++s)
            st.qf[s] = frag_global((const T*)a.q + (live ? qrows.at(row) : 0) + s * 16 + h * 8, live && s * 16 + h * 8 < a.D);
#pragma unroll
        for (int i = 0; i < DT; ++i) st.acc[i] = zero16();
        st.base = -3.0e38f;
        st.l = 0.f;
        const int nfull = jall / BN;        // steps whose keys are all there and all seen: no mask, and loaded while the one before computes
        if (nfull > 0) {
            __syncthreads();
            dk.load(k, a.k_st, at_lds);
            dv.load(v, a.v_st, at_lds + TB);
            for (int t = 0; t < nfull; ++t) {
                char* now = lds + (t & 1) * 2 * TB;
                wait_loads<0>();
                __syncthreads();            // tile t is there, and nobody reads the other buffer any more
                if (t + 1 < nfull) {
                    const unsigned next = at_lds + ((t + 1) & 1) * 2 * TB;
                    dk.load(k + (long long)(t + 1) * BN * a.k_st, a.k_st, next);
                    dv.load(v + (long long)(t + 1) * BN * a.v_st, a.v_st, next + TB);
                }
                st.template step<false>(now, now + TB, lane, c2, BN);
            }
        }
        for (int k0 = nfull * BN; k0 < jend; k0 += BN) {
            __syncthreads();
            stage<T, DP, BN, false>(lds, k + (long long)k0 * a.k_st, sk.n - k0, a.D, [&](int r) { return (long long)r * a.k_st; });
            bool bad = stage<T, DP, BN, true>(lds + TB, v + (long long)k0 * a.v_st, sk.n - k0, a.D, [&](int r) { return (long long)r * a.v_st; });
            bad = __syncthreads_or(bad);
            if (k0 < jwave) st.template step<true>(lds, lds + TB, lane, c2, jmax - k0);
            if (bad) add_nonfinite<T, DT>(st.acc, v + (long long)k0 * a.v_st, a.v_st, min(jmax - k0, BN), a.D, h);
        }
        const float l = st.l + __shfl_xor(st.l, 32, 64);
        const float inv = one_over(l, jmax);
        if (live) {
            const int t = row / a.G, head = kv * a.G + row - t * a.G;
            const long long at = (sq.begin + t) * a.Hq + head;
            T* o = out + at * a.D;
#pragma unroll
            for (int d = 0; d < DT; ++d) store_cols(o, st.acc[d], d, h, a.D, inv);
            if (a.stats && h == 0) a.stats[at] = make_float2(st.base, inv);
            if (a.lse && h == 0) a.lse[at] = inv == 0.f ? -INFINITY : st.base * LN2 + logf(l);
        }
    }
}

// ------------------------------------------------------------------------------------- forward for few rows, split over the keys
// With few rows (one new token of each request: the heads of one group) the keys are what has to be read, once, and nothing else
// counts.  A wave is a workgroup here: it takes 32 rows and a chunk of keys in blocks of 32, with two tiles of its own that the next
// block's loads fill while it computes (no barrier: a wave waits for its own loads), and the chunks' results meet in k_attn_join.
// Bound by HBM: 24 requests of 1 .. 32768 keys, 8 key heads of 128 (2.03 GB) in 403 to 440 us = 4.6 to 5.0 TB/s, where a copy runs at 5.1.  Workgroups of 2
// or 4 waves that join in LDS were 15 to 50 % slower on short caches (32768 keys of one request: 46 and 60 us against 40 of this kernel then).
template <typename T, int DP>
struct FewCfg {
    static constexpr int TB = 32 * DP * (int)sizeof(T), LDS = 4 * TB;
};

struct Few {
    int tiles, splits, chunk;       // row tiles of a pair, chunks of the longest sequence, keys of a chunk
    float* part;                    // [splits, Tq * Hq, D] unnormalised results, and
    float2* pstat;                  // [splits, Tq * Hq] their bases and sums; unused with one split
    unsigned first_rest;
};

template <typename T, int DP, bool FINE>
__global__ __launch_bounds__(64, (FewCfg<T, DP>::LDS >= 32768 ? 1 : 2)) void k_attn_few(Attn a, Few f) {
    typedef Tile<T, DP> L;
    constexpr int KS = DP / 16, DT = DP / 32, TB = FewCfg<T, DP>::TB;
    __shared__ __attribute__((aligned(1024))) char mine[FewCfg<T, DP>::LDS];       // two tiles of keys and values
    const int lane = threadIdx.x, h = lane >> 5;
    T* out = (T*)a.out;
    if (blockIdx.x >= f.first_rest) {
        const Rest z = rest(a.cu_q, a.B, a.Tq);
        for (long long i = (long long)(blockIdx.x - f.first_rest) * 8 + (lane >> 3); i < z.n * a.Hq; i += (long long)(gridDim.x - f.first_rest) * 8) {
            const long long r = z.row(i / a.Hq) * a.Hq + i % a.Hq;
            zero_row(out + r * a.D, a.D, threadIdx.x & 7, 8);
            if (a.lse && (threadIdx.x & 7) == 0) a.lse[r] = -INFINITY;
        }
        return;
    }
    const Place pl = place(blockIdx.x, a.B * a.Hk * f.splits, f.tiles);
    if (pl.tile < 0) return;
    // the key heads of a chunk are neighbours: their rows lie side by side in memory
    const int chunk = pl.pair / a.Hk, kv = pl.pair - chunk * a.Hk, b = chunk / f.splits, split = chunk - b * f.splits;
    const Span sq = span(a.cu_q, nullptr, b, a.Tq), sk = span(a.cu_k, a.len_k, b, a.Tk);
    const int R = sq.n * a.G;
    if ((long long)pl.tile * 32 >= R) return;
    const Rows qrows{sq.begin, a.q_st, a.q_sh, a.G, kv * a.G};
    const T *k = (const T*)a.k + sk.begin * a.k_st + kv * a.k_sh, *v = (const T*)a.v + sk.begin * a.v_st + kv * a.v_sh;
    const float c2 = a.scale * LOG2E;
    const Dma<T, DP, 32, 64> dk(a.k_st, a.D), dv(a.v_st, a.D);
    const unsigned at_lds = lds_at(mine);
    for (long long rr = (long long)pl.tile * 32; rr < R; rr += (long long)f.tiles * 32) {
        const int r0 = (int)rr, row = r0 + (lane & 31);
        const bool live = row < R;
        const int jmax = live ? seen_keys(row / a.G, sq.n, sk.n, a.causal) : 0;
        const int last = min(r0 + 32, R) - 1;
        const int jend = seen_keys(last / a.G, sq.n, sk.n, a.causal), jall = seen_keys(r0 / a.G, sq.n, sk.n, a.causal);
        if (f.splits > 1 && (long long)split * f.chunk >= jend && (split > 0 || jend > 0)) continue;      // (chunk 0 answers for a row without keys)
        if (a.D < DP) {
            for (int i = lane; i < 4 * TB / 16; i += 64) reinterpret_cast<uint4*>(mine)[i] = make_uint4(0, 0, 0, 0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        FwdState<T, DP, 32> st;
#pragma unroll
        for (int s = 0; s < KS; ++s)
            st.qf[s] = frag_global((const T*)a.q + (live ? qrows.at(row) : 0) + s * 16 + h * 8, live && s * 16 + h * 8 < a.D);
        // With FINE an infinity among the values, multiplied by a weight's rest that is zero or negative, would come out as NaN: where a result is
        // not finite the keys are gone over once more, each block checked as those at the border are.
        for (bool checked = false;; checked = true) {
#pragma unroll
            for (int i = 0; i < DT; ++i) st.acc[i] = zero16();
            st.base = -3.0e38f;
            st.l = 0.f;
            for (long long c0 = (long long)split * f.chunk; c0 < jend; c0 += (long long)f.splits * f.chunk) {
                const int begin = (int)c0, end = (int)(c0 + f.chunk < jend ? c0 + f.chunk : jend);
                const int full = !checked && min(end, jall) >= begin ? (min(end, jall) - begin) / 32 : 0;       // blocks that need no mask
                int blk = 0, buf = 0;
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (blk < full) {
                    dk.load(k + (long long)(begin + blk * 32) * a.k_st, a.k_st, at_lds);
                    dv.load(v + (long long)(begin + blk * 32) * a.v_st, a.v_st, at_lds + TB);
                    wait_loads<0>();        // (for the rows' own loads too, which the loop would otherwise wait for)
                }
                for (; blk < full; ++blk, buf ^= 1) {
                    char* now = mine + buf * 2 * TB;
                    const unsigned next = at_lds + (buf ^ 1) * 2 * TB;
                    // what was read of the other buffer has arrived; then its new loads, and the wait for all but those
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    if (blk + 1 < full) {
                        dk.load(k + (long long)(begin + (blk + 1) * 32) * a.k_st, a.k_st, next);
                        dv.load(v + (long long)(begin + (blk + 1) * 32) * a.v_st, a.v_st, next + TB);
                        wait_loads<2 * Dma<T, DP, 32, 64>::N>();
                    } else {
                        wait_loads<0>();
                    }
                    st.template step<false, FINE>(now, now + TB, lane, c2, 32);
                }
                for (int i = full; begin + i * 32 < end; ++i) {
                    const int k0 = begin + i * 32;
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    stage<T, DP, 32, false, 64>(mine, k + (long long)k0 * a.k_st, sk.n - k0, a.D, [&](int r) { return (long long)r * a.k_st; });
                    const bool bad = __any(stage<T, DP, 32, true, 64>(mine + TB, v + (long long)k0 * a.v_st, sk.n - k0, a.D, [&](int r) { return (long long)r * a.v_st; }));
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    st.template step<true, FINE>(mine, mine + TB, lane, c2, min(jmax, end) - k0);
                    if (bad) add_nonfinite<T, DT>(st.acc, v + (long long)k0 * a.v_st, a.v_st, min(min(jmax, end) - k0, 32), a.D, h);
                }
            }
            if (!FINE || checked) break;
            float odd = 0.f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) odd = fmaf(st.acc[d][i], 0.f, odd);
            if (!__any(odd != 0.f)) break;
        }
        const float l = st.l + __shfl_xor(st.l, 32, 64);
        if (!live) continue;
        const int t = row / a.G;
        const long long at = (sq.begin + t) * a.Hq + kv * a.G + (row - t * a.G);
        if (f.splits > 1) {
            const long long to = (long long)split * a.Tq * a.Hq + at;
#pragma unroll
            for (int d = 0; d < DT; ++d) store_cols(f.part + to * a.D, st.acc[d], d, h, a.D, 1.f);
            if (h == 0) f.pstat[to] = make_float2(st.base, l);
        } else {
            const float inv = one_over(l, jmax);
#pragma unroll
            for (int d = 0; d < DT; ++d) store_cols(out + at * a.D, st.acc[d], d, h, a.D, inv);
            if (a.stats && h == 0) a.stats[at] = make_float2(st.base, inv);
            if (a.lse && h == 0) a.lse[at] = inv == 0.f ? -INFINITY : st.base * LN2 + logf(l);
        }
    }
}

// The chunks' results of a row: 32 lanes have four elements each, eight groups of lanes take every eighth chunk; the groups' sums meet in
// a fixed order.  One workgroup per row, so that a single request over many chunks is not read by a handful of waves.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_join(Attn a, Few f) {
    __shared__ float4 sums[8][32];
    __shared__ float part_sum[8];
    const int b = blockIdx.y, lane = threadIdx.x & 31, grp = threadIdx.x >> 5, d = lane * 4;
    const Span sq = span(a.cu_q, nullptr, b, a.Tq), sk = span(a.cu_k, a.len_k, b, a.Tk);
    T* out = (T*)a.out;
    const long long all = a.Tq * a.Hq;
    for (long long row = blockIdx.x; row < (long long)sq.n * a.Hq; row += gridDim.x) {
        const int head = (int)(row % a.Hq), t = (int)(row / a.Hq);
        const long long at = (sq.begin + t) * a.Hq + head;
        // the keys of this row's tile, as k_attn_few counted them
        const int r = t * a.G + head % a.G, last = min((r / 32 + 1) * 32, sq.n * a.G) - 1;
        const int jend = seen_keys(last / a.G, sq.n, sk.n, a.causal);
        const int n = jend > 0 ? min(f.splits, (jend - 1) / f.chunk + 1) : 1;
        float base = -3.0e38f;
        for (int s = threadIdx.x & 63; s < n; s += 64) base = fmaxf(base, f.pstat[s * all + at].x);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) base = fmaxf(base, __shfl_xor(base, o, 64));
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
#pragma unroll 4
        for (int s = grp; s < n; s += 8) {
            const float2 ps = f.pstat[s * all + at];
            const float4 x = d < a.D ? *reinterpret_cast<const float4*>(f.part + (s * all + at) * a.D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            const float e = ps.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ps.x - base);        // (a chunk of which the row saw nothing holds zeros)
            o.x += x.x * e; o.y += x.y * e; o.z += x.z * e; o.w += x.w * e;
            sum += ps.y * e;
        }
        sums[grp][lane] = o;
        if (lane == 0) part_sum[grp] = sum;
        __syncthreads();
        if (grp == 0) {
#pragma unroll
            for (int g = 1; g < 8; ++g) {
                const float4 x = sums[g][lane];
                o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
                sum += part_sum[g];
            }
            const float inv = one_over(sum, seen_keys(t, sq.n, sk.n, a.causal));
            if (d < a.D) {
                if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(out + at * a.D + d) = make_uint2(pack2(o.x * inv, o.y * inv), pack2(o.z * inv, o.w * inv));
                else *reinterpret_cast<float4*>(out + at * a.D + d) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
            }
            if (lane == 0 && a.stats) a.stats[at] = make_float2(base, inv);
            if (lane == 0 && a.lse) a.lse[at] = inv == 0.f ? -INFINITY : base * LN2 + logf(sum);
        }
        __syncthreads();
    }
}

// -------------------------------------------------------------------------------------------------- gradient of q (and D)
// D_i = go_i o_i comes from the forward's result -- rounded, which costs a row that sees n keys about 2^-9 / sqrt(n) of its dS beside the
// 2^-9 of dS's own rounding.  Where no row of a tile sees more than EXACT_D keys, D is summed as sum_j p_ij (go_i v_j) instead, in a first
// sweep over the keys (32 prompts of up to 32 tokens: the error of gq and gk against 64 bits falls from 3.1e-3 to 2.4e-3).
constexpr int EXACT_D = 128;
// The forward's layout with two scores per key: s = q k and go v.  The weights keep the forward's exponent base and stay unnormalised;
// the row's 1 / sum goes into the result with the scale, so what the base lost in rounding cancels as it does in the forward.
template <typename T, int DP>
struct GqCfg {
    static constexpr int BN = sizeof(T) * DP > 256 ? 32 : 64;
    static constexpr bool FINE = DP <= 32;      // (rest_of())
};

template <typename T, int DP, int BN>
struct GqState {
    typedef Tile<T, DP> L;
    static constexpr int KS = DP / 16, DT = DP / 32;
    Frag<T> qf[KS], gf[KS];
    f32x16 acc[DT];
    float base, delta, sum;

    // the keys first .. end - 1 that are not finite, and that the steps took for zeros, into the row's gradient in memory
    __device__ __forceinline__ void add_spoilt(T* out, float mul, const T* q, const T* go, const T* k, long long k_st, const T* v, long long v_st, int first, int end, int D, int h,
                                               float c2) const {
#pragma unroll 1
        for (int j = first; j < end; ++j)
            if (spoils(k + j * k_st, D) &&
                add_to_row(out, __builtin_amdgcn_exp2f(fmaf(dot(q, k + j * k_st, D), c2, -base)) * (dot(go, v + j * v_st, D) - delta) * mul, k + j * k_st, D, h, false))
                return;
    }
    template <bool MASK, bool SUM = false, bool FINE = false>
    __device__ __forceinline__ void step(const char* lk, const char* lv, int lane, float c2, int left) {
        const int h = lane >> 5;
#pragma unroll
        for (int sub = 0; sub < BN / 32; ++sub) {
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                s = mma(L::row_frag(lk, sub * 32 + (lane & 31), i, h), qf[i], s);
                dp = mma(L::row_frag(lv, sub * 32 + (lane & 31), i, h), gf[i], dp);
            }
            float ds[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                ds[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c2, -base)) * (dp[i] - delta);
                if (MASK && sub * 32 + reg_row(i, h) >= left) ds[i] = 0.f;
            }
            if (SUM) {          // delta is 0: ds is p (go v), summed for D
#pragma unroll
                for (int i = 0; i < 16; ++i) sum += ds[i];
                continue;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                Frag<T> f, r;
                frag_of(f, ds + 8 * t);
                if (FINE) rest_of(r, f, ds + 8 * t);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const Frag<T> kf = L::col_frag(lk, sub * 32 + 16 * t, d, lane);
                    acc[d] = mma(kf, f, acc[d]);
                    if (FINE && sizeof(T) == 2) acc[d] = mma(kf, r, acc[d]);
                }
            }
        }
    }
};

template <typename T, int DP, bool LISTED>
__global__ __launch_bounds__(256, (sizeof(T) * DP > 256 ? 1 : sizeof(T) * DP <= 64 ? 3 : 2)) void k_attn_gq(Attn a, int tiles, unsigned first_rest) {
    typedef Tile<T, DP> L;
    constexpr int BN = GqCfg<T, DP>::BN, TB = BN * L::ROWB;
    constexpr int KS = DP / 16, DT = DP / 32;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TB];
    __shared__ int odd[4];          // a wave's: a key at the border was not finite (kept here, where it takes no register from the loop)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    T* gq = (T*)a.gq;
    if (blockIdx.x >= first_rest) {
        const Rest z = rest(a.cu_q, a.B, a.Tq);
        for (long long i = (long long)(blockIdx.x - first_rest) * 32 + (threadIdx.x >> 3); i < z.n * a.Hq; i += (long long)(gridDim.x - first_rest) * 32)
            zero_row(gq + (z.row(i / a.Hq) * a.Hq + i % a.Hq) * a.D, a.D, threadIdx.x & 7, 8);
        return;
    }
    const Place pl = LISTED ? listed<BM>(blockIdx.x, a.cu_q, a.B, a.Hk, a.G, a.Tq) : place(blockIdx.x, a.B * a.Hk, tiles);
    if (pl.tile < 0) return;
    const int b = pl.pair / a.Hk, kv = pl.pair - b * a.Hk;
    const Span sq = span(a.cu_q, nullptr, b, a.Tq), sk = span(a.cu_k, nullptr, b, a.Tk);
    const int R = sq.n * a.G;
    if ((long long)pl.tile * BM >= R) return;
    const Rows qrows{sq.begin, a.q_st, a.q_sh, a.G, kv * a.G}, grows{sq.begin, a.go_st, a.go_sh, a.G, kv * a.G};
    const T *k = (const T*)a.k + sk.begin * a.k_st + kv * a.k_sh, *v = (const T*)a.v + sk.begin * a.v_st + kv * a.v_sh;
    const float c2 = a.scale * LOG2E;
    const Dma<T, DP, BN> dk(a.k_st, a.D), dv(a.v_st, a.D);
    const unsigned at_lds = lds_at(lds) + wave * 1024;
    if (a.D < DP) {
        for (int i = threadIdx.x; i < 4 * TB / 16; i += 256) reinterpret_cast<uint4*>(lds)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    for (long long rr = (long long)pl.tile * BM; rr < R; rr += (long long)tiles * BM) {
        const int r0 = (int)rr;
        const int row = r0 + wave * 32 + (lane & 31);
        const bool live = row < R;
        const int tok = live ? row / a.G : 0;
        const long long at = live ? (sq.begin + tok) * a.Hq + kv * a.G + (row - tok * a.G) : 0;     // row of [Tq, Hq]
        const int jmax = live ? seen_keys(tok, sq.n, sk.n, a.causal) : 0;
        const int last = min(r0 + BM, R) - 1;
        const int jend = seen_keys(last / a.G, sq.n, sk.n, a.causal);
        const int jall = seen_keys(r0 / a.G, sq.n, sk.n, a.causal);
        const int jwave = r0 + wave * 32 < R ? seen_keys(min(r0 + wave * 32 + 31, last) / a.G, sq.n, sk.n, a.causal) : 0;
        if (lane == 0) odd[wave] = 0;
        GqState<T, DP, BN> st;
        const float2 stat = live ? a.stats[at] : make_float2(0.f, 0.f);
        st.base = stat.x;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = s * 16 + h * 8;
            const bool on = live && d < a.D;
            st.qf[s] = frag_global((const T*)a.q + (live ? qrows.at(row) : 0) + d, on);
            st.gf[s] = frag_global((const T*)a.go + (live ? grows.at(row) : 0) + d, on);
        }
        float delta = 0.f;
        if (jend <= EXACT_D) {
            st.delta = st.sum = 0.f;
            for (int k0 = 0; k0 < jend; k0 += BN) {
                __syncthreads();
                stage<T, DP, BN, false>(lds, k + (long long)k0 * a.k_st, sk.n - k0, a.D, [&](int r) { return (long long)r * a.k_st; });
                stage<T, DP, BN, false>(lds + TB, v + (long long)k0 * a.v_st, sk.n - k0, a.D, [&](int r) { return (long long)r * a.v_st; });
                __syncthreads();
                if (k0 < jwave) st.template step<true, true>(lds, lds + TB, lane, c2, jmax - k0);
            }
            delta = st.sum * stat.y;
        } else {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = s * 16 + h * 8;
                if (live && d < a.D) {
                    Raw8<T> x, y;
                    float fx[8], fy[8];
                    x.load((const T*)a.o + at * a.D + d);
                    y.load((const T*)a.go + grows.at(row) + d);
                    x.get(fx);
                    y.get(fy);
#pragma unroll
                    for (int j = 0; j < 8; ++j) delta += fx[j] * fy[j];
                }
            }
        }
        st.delta = delta + __shfl_xor(delta, 32, 64);
        if (live && h == 0) {
            const long long all = a.Tq * a.Hq;
            float* to = a.rowstat + ((long long)kv * a.Tq + sq.begin) * a.G + row;        // the rows of a pair lie in order
            to[0] = sizeof(T) == 4 ? stat.x : stat.x - __builtin_amdgcn_logf(stat.y);
            to[all] = st.delta;
            if (sizeof(T) == 4) to[2 * all] = stat.y;
        }
#pragma unroll
        for (int i = 0; i < DT; ++i) st.acc[i] = zero16();
        const int nfull = jall / BN;
        if (nfull > 0) {
            __syncthreads();
            dk.load(k, a.k_st, at_lds);
            dv.load(v, a.v_st, at_lds + TB);
            for (int t = 0; t < nfull; ++t) {
                char* now = lds + (t & 1) * 2 * TB;
                wait_loads<0>();
                __syncthreads();
                if (t + 1 < nfull) {
                    const unsigned next = at_lds + ((t + 1) & 1) * 2 * TB;
                    dk.load(k + (long long)(t + 1) * BN * a.k_st, a.k_st, next);
                    dv.load(v + (long long)(t + 1) * BN * a.v_st, a.v_st, next + TB);
                }
                st.template step<false, false, GqCfg<T, DP>::FINE>(now, now + TB, lane, c2, BN);
            }
        }
        for (int k0 = nfull * BN; k0 < jend; k0 += BN) {
            __syncthreads();
            bool bad = stage<T, DP, BN, true>(lds, k + (long long)k0 * a.k_st, sk.n - k0, a.D, [&](int r) { return (long long)r * a.k_st; });
            stage<T, DP, BN, false>(lds + TB, v + (long long)k0 * a.v_st, sk.n - k0, a.D, [&](int r) { return (long long)r * a.v_st; });
            bad = __syncthreads_or(bad);
            if (bad) {
                if (lane == 0) odd[wave] = 1;
                clear_spoilt<T, DP, 256>(lds, k + (long long)k0 * a.k_st, a.k_st, min(sk.n - k0, BN), a.D);
                __syncthreads();
            }
            if (k0 < jwave) st.template step<true, false, GqCfg<T, DP>::FINE>(lds, lds + TB, lane, c2, jmax - k0);
        }
        if (live) {
            T* o = gq + at * a.D;
            const float mul = a.scale * stat.y;
#pragma unroll
            for (int d = 0; d < DT; ++d) store_cols(o, st.acc[d], d, h, a.D, mul);
            if (odd[wave]) st.add_spoilt(o, mul, (const T*)a.q + qrows.at(row), (const T*)a.go + grows.at(row), k, a.k_st, v, a.v_st, jall / BN * BN, jmax, a.D, h, c2);
        }
    }
}

// --------------------------------------------------------------------------------------------- gradients of k and v
// One key per lane, the rows that see it in registers; rows pass through LDS, so no sum leaves the workgroup and none is atomic.
// For 128 elements of 16 bits the value rows stay in LDS instead of registers: two waves share a SIMD's registers then.
template <typename T, int DP>
struct GkvCfg {
    static constexpr int BR = sizeof(T) * DP >= 256 ? 32 : 64;         // rows of a step
    static constexpr bool V_LDS = sizeof(T) * DP >= 256;
    static constexpr int WAVES = sizeof(T) * DP > 256 ? 1 : 2;         // per SIMD
};

// What the steps left out of the rows first .. end - 1, which see a key: queries and gradients of the result that are not finite, into the key's
// gradients in memory.  st: the statistics of row 0 (rare path)
template <typename T>
__device__ void add_spoilt(T* gk, T* gv, const Attn& a, const Rows& qrows, const Rows& grows, const T* k, const T* v, const float* st, long long pitch, int first, int end, int h) {
#pragma unroll 1
    for (int r = first; r < end; ++r) {
        const T *q = (const T*)a.q + qrows.at(r), *go = (const T*)a.go + grows.at(r);
        if (!spoils(q, a.D) && !spoils(go, a.D)) continue;
        const float p = __builtin_amdgcn_exp2f(fmaf(dot(q, k, a.D), a.scale * LOG2E, -st[r])) * (sizeof(T) == 4 ? st[2 * pitch + r] : 1.f);
        const bool all_v = add_to_row(gv, p, go, a.D, h, true), all_k = add_to_row(gk, p * (dot(go, v, a.D) - st[pitch + r]) * a.scale, q, a.D, h, false);
        if (all_v && all_k) return;
    }
}

// The rows of a step (BR of them, STEP to the next) of q and go into LDS by NT threads.  EVEN: the heads of a group divide a step, so a lane's rows stay where they are
// from step to step and only the wave's address moves.  Otherwise each lane follows its rows: a step is adv_t tokens and adv_g heads, one
// token more where the head leaves the group.
template <typename T, int DP, int BR, bool EVEN, int NT = 256, int STEP = BR>
struct RowDma {
    typedef Tile<T, DP> L;
    static constexpr int RPI = NT / L::CPR, N = (BR + RPI - 1) / RPI;
    static_assert(BR % RPI == 0 || N == 1, "whole rounds");
    const T *q, *go;
    unsigned oq[N], og[N];
    bool on[N];
    __device__ __forceinline__ RowDma(const T* q0, const T* go0, const Attn& a, int r0) : q(q0 + r0 / a.G * a.q_st), go(go0 + r0 / a.G * a.go_st) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = i * RPI + (int)threadIdx.x % NT / L::CPR, c = ((threadIdx.x % L::CPR) ^ L::f(row)) * L::EPC, t = row / a.G, g = row - t * a.G;
            on[i] = c < a.D && row < BR;
            oq[i] = (unsigned)((t * a.q_st + g * a.q_sh + c) * (long long)sizeof(T));
            og[i] = (unsigned)((t * a.go_st + g * a.go_sh + c) * (long long)sizeof(T));
        }
    }
    __device__ __forceinline__ void advance(const Attn& a) {
        q += STEP / a.G * a.q_st;
        go += STEP / a.G * a.go_st;
#pragma unroll
        for (int i = 0; i < N; ++i) asm volatile("" : "+v"(oq[i]), "+v"(og[i]));        // (registers, not scratch: a reload waits for the loads)
    }
    __device__ __forceinline__ void load(unsigned lq, unsigned lg) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (on[i]) {
                load_to_lds(q, oq[i], lq + i * NT * 16);
                load_to_lds(go, og[i], lg + i * NT * 16);
            }
    }
};
template <typename T, int DP, int BR, int NT, int STEP>
struct RowDma<T, DP, BR, false, NT, STEP> {
    typedef Tile<T, DP> L;
    static constexpr int RPI = NT / L::CPR, N = (BR + RPI - 1) / RPI;
    const T *q[N], *go[N];
    int g[N];
    bool on[N];
    __device__ __forceinline__ RowDma(const T* q0, const T* go0, const Attn& a, int r0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = i * RPI + (int)threadIdx.x % NT / L::CPR, c = ((threadIdx.x % L::CPR) ^ L::f(row)) * L::EPC;
            const int tok = (r0 + row) / a.G;
            on[i] = c < a.D && row < BR;
            g[i] = r0 + row - tok * a.G;
            q[i] = q0 + tok * a.q_st + g[i] * a.q_sh + c;
            go[i] = go0 + tok * a.go_st + g[i] * a.go_sh + c;
        }
    }
    __device__ __forceinline__ void advance(const Attn& a) {
        const int adv_t = STEP / a.G, adv_g = STEP - adv_t * a.G;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            g[i] += adv_g;
            const bool over = g[i] >= a.G;
            q[i] += adv_t * a.q_st + adv_g * a.q_sh + (over ? a.q_st - a.G * a.q_sh : 0);
            go[i] += adv_t * a.go_st + adv_g * a.go_sh + (over ? a.go_st - a.G * a.go_sh : 0);
            g[i] -= over ? a.G : 0;
        }
    }
    __device__ __forceinline__ void load(unsigned lq, unsigned lg) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (on[i]) {
                load_to_lds(q[i], lq + i * NT * 16);
                load_to_lds(go[i], lg + i * NT * 16);
            }
    }
};

// One step of 32 rows for 32 keys: what both kernels for gk and gv compute.  lq, lg: the rows' tiles; lvw: the wave's value rows where they
// are in LDS; st: exponent base, D and (32 bits) 1 / sum of the rows, `pitch` apart.  Rows r0 .. are seen from row `from` to `end`.
template <typename T, int DP, bool V_LDS>
struct GkvState {
    typedef Tile<T, DP> L;
    static constexpr int KS = DP / 16, DT = DP / 32;
    static constexpr bool F32 = sizeof(T) == 4;
    Frag<T> kf[KS], vf[V_LDS ? 1 : KS];
    f32x16 ak[DT], av[DT];

    __device__ __forceinline__ void begin(const T* k, const T* v, bool live, int D, int h) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = s * 16 + h * 8;
            kf[s] = frag_global(k + d, live && d < D);
            if (!V_LDS) vf[s] = frag_global(v + d, live && d < D);
        }
#pragma unroll
        for (int i = 0; i < DT; ++i) ak[i] = zero16(), av[i] = zero16();
    }
    template <bool MASK, bool FINE = false>
    __device__ __forceinline__ void step(const char* lq, const char* lg, const char* lvw, const float* st, int pitch, int lane, float c2, int r0, int from, int end) {
        const int h = lane >> 5;
        f32x16 s = zero16(), dp = zero16();
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            s = mma(L::row_frag(lq, lane & 31, i, h), kf[i], s);
            if constexpr (V_LDS) dp = mma(L::row_frag(lg, lane & 31, i, h), L::row_frag(lvw, lane & 31, i, h), dp);
            else dp = mma(L::row_frag(lg, lane & 31, i, h), vf[i], dp);
            // (left alone, the compiler reads every operand ahead and spills; a reload in the loop waits for the tiles' loads)
            if (V_LDS && i % 2 == 1) __builtin_amdgcn_sched_barrier(0);
        }
        Frag<T> pf[2], df[2], pr[2], dr[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float ba[8], de[8], in[8], p[8], ds[8];
#pragma unroll
            for (int q4 = 0; q4 < 2; ++q4) {
                const int r4 = 16 * t + 8 * q4 + 4 * h;
                *reinterpret_cast<float4*>(ba + 4 * q4) = *reinterpret_cast<const float4*>(st + r4);
                *reinterpret_cast<float4*>(de + 4 * q4) = *reinterpret_cast<const float4*>(st + pitch + r4);
                if (F32) *reinterpret_cast<float4*>(in + 4 * q4) = *reinterpret_cast<const float4*>(st + 2 * pitch + r4);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = 8 * t + e, r = r0 + reg_row(i, h);
                p[e] = __builtin_amdgcn_exp2f(fmaf(s[i], c2, -ba[e]));
                if (F32) p[e] *= in[e];
                ds[e] = p[e] * (dp[i] - de[e]);
                if (MASK && !(r >= from && r < end)) p[e] = ds[e] = 0.f;
            }
            frag_of(pf[t], p);
            frag_of(df[t], ds);
            if (FINE) rest_of(pr[t], pf[t], p), rest_of(dr[t], df[t], ds);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                // (left alone, the compiler keeps five reloads in the loop: heads of 128, 5 prompts of 601 .. 5184: 1330 -> 1250 us)
                if (V_LDS && !F32 && d == 1) __builtin_amdgcn_sched_barrier(0);
                const Frag<T> gf = L::col_frag(lg, 16 * t, d, lane), qf = L::col_frag(lq, 16 * t, d, lane);
                av[d] = mma(gf, pf[t], av[d]);
                ak[d] = mma(qf, df[t], ak[d]);
                if (FINE && sizeof(T) == 2) av[d] = mma(gf, pr[t], av[d]), ak[d] = mma(qf, dr[t], ak[d]);
            }
    }
};

template <typename T, int DP, bool EVEN, bool LISTED>
__global__ __launch_bounds__(256, (GkvCfg<T, DP>::WAVES)) void k_attn_gkv(Attn a, int tiles, unsigned first_rest) {
    typedef Tile<T, DP> L;
    typedef GkvCfg<T, DP> C;
    constexpr int DT = DP / 32, BK = 128, BR = C::BR, TB = BR * L::ROWB;
    constexpr bool F32 = sizeof(T) == 4;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TB + (C::V_LDS ? BK * L::ROWB : 0)];
    __shared__ __attribute__((aligned(1024))) float stat[2][F32 ? 3 : 2][BR];
    __shared__ int odd[4];          // a wave's: a row at the border was not finite (kept here, where it takes no register from the loop)
    char* lvt = lds + 4 * TB;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    T *gk = (T*)a.gk, *gv = (T*)a.gv;
    if (blockIdx.x >= first_rest) {
        const Rest z = rest(a.cu_k, a.B, a.Tk);
        for (long long i = (long long)(blockIdx.x - first_rest) * 32 + (threadIdx.x >> 3); i < z.n * a.Hk; i += (long long)(gridDim.x - first_rest) * 32) {
            const long long r = z.row(i / a.Hk) * a.Hk + i % a.Hk;
            zero_row(gk + r * a.D, a.D, threadIdx.x & 7, 8);
            zero_row(gv + r * a.D, a.D, threadIdx.x & 7, 8);
        }
        return;
    }
    const Place pl = LISTED ? listed<BK>(blockIdx.x, a.cu_k, a.B, a.Hk, 1, a.Tk) : place(blockIdx.x, a.B * a.Hk, tiles);
    if (pl.tile < 0) return;
    const int tile = LISTED ? pl.tile : tiles - 1 - pl.tile;       // the first keys have the most rows
    const int b = pl.pair / a.Hk, kv = pl.pair - b * a.Hk;
    const Span sq = span(a.cu_q, nullptr, b, a.Tq), sk = span(a.cu_k, nullptr, b, a.Tk);
    if ((long long)tile * BK >= sk.n) return;
    const int R = sq.n * a.G;
    const Rows qrows{sq.begin, a.q_st, a.q_sh, a.G, kv * a.G}, grows{sq.begin, a.go_st, a.go_sh, a.G, kv * a.G};
    const T *k = (const T*)a.k + sk.begin * a.k_st + kv * a.k_sh, *v = (const T*)a.v + sk.begin * a.v_st + kv * a.v_sh;
    const T *q0 = (const T*)a.q + sq.begin * a.q_st + (long long)kv * a.G * a.q_sh, *g0 = (const T*)a.go + sq.begin * a.go_st + (long long)kv * a.G * a.go_sh;
    const float c2 = a.scale * LOG2E;
    const long long all = a.Tq * a.Hq;
    const unsigned at_lds = lds_at(lds) + wave * 1024, at_stat = lds_at(stat) + wave * BR * 4;      // (wave i brings the i-th statistic)
    const float* rowstat = a.rowstat + ((long long)kv * a.Tq + sq.begin) * a.G;
    if (a.D < DP) {
        for (int i = threadIdx.x; i < 4 * TB / 16; i += 256) reinterpret_cast<uint4*>(lds)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    for (long long kk = (long long)tile * BK; kk < sk.n; kk += (long long)tiles * BK) {
        const int k0 = (int)kk;
        const int key = k0 + wave * 32 + (lane & 31);
        const bool live = key < sk.n;
        if (lane == 0) odd[wave] = 0;
        GkvState<T, DP, C::V_LDS> st;
        st.begin(k + (live ? key * a.k_st : 0), v + (live ? key * a.v_st : 0), live, a.D, h);
        __syncthreads();
        if (C::V_LDS) stage<T, DP, BK, false>(lvt, v + (long long)k0 * a.v_st, sk.n - k0, a.D, [&](int r) { return (long long)r * a.v_st; });
        // rows before first see no key of the tile; from r_all on they see all of them; from r_key on, this lane's
        const auto first_row = [&](int j) {
            const long long t = a.causal ? (long long)j - (sk.n - sq.n) : 0;
            return (t < 0 ? 0 : t > sq.n ? sq.n : (int)t) * a.G;
        };
        const int first = first_row(k0), r_all = first_row(min(k0 + BK, sk.n) - 1), r_key = live ? first_row(key) : R;

        const auto step = [&](auto mask, int buf, int r0) {
#pragma unroll
            for (int sub = 0; sub < BR / 32; ++sub)
                st.template step<decltype(mask)::value>(lds + buf * 2 * TB + sub * 32 * L::ROWB, lds + buf * 2 * TB + TB + sub * 32 * L::ROWB, lvt + wave * 32 * L::ROWB,
                                                        &stat[buf][0][sub * 32], BR, lane, c2, r0 + sub * 32, r_key, R);
        };
        const auto border = [&](int r0) {
            __syncthreads();
            if ((int)threadIdx.x < BR) {
                const bool on = r0 + (int)threadIdx.x < R;
#pragma unroll
                for (int i = 0; i < (F32 ? 3 : 2); ++i) stat[0][i][threadIdx.x] = on ? rowstat[i * all + r0 + threadIdx.x] : 0.f;
            }
            bool bad = stage<T, DP, BR, true>(lds, (const T*)a.q, R - r0, a.D, [&](int r) { return qrows.at(r0 + r); });
            bad |= stage<T, DP, BR, true>(lds + TB, (const T*)a.go, R - r0, a.D, [&](int r) { return grows.at(r0 + r); });
            if (__syncthreads_or(bad) && lane == 0) odd[wave] = 1;
            step(std::true_type{}, 0, r0);
        };
        int r0 = first;
        for (; r0 < R && r0 < r_all; r0 += BR) border(r0);
        const int nfull = r0 < R ? (R - r0) / BR : 0;
        if (nfull > 0) {
            RowDma<T, DP, BR, EVEN> dma(q0, g0, a, r0);
            const float* sp = rowstat + wave * all;
            const bool son = wave < (F32 ? 3 : 2) && lane < BR;
            __syncthreads();
            dma.load(at_lds, at_lds + TB);
            if (son) word_to_lds(sp + r0, lane * 4, at_stat);
            const auto full = [&](auto buf, int t) {
                constexpr int NOW = decltype(buf)::value, NEXT = 1 - NOW;
                wait_loads<0>();
                __syncthreads();
                if (t + 1 < nfull) {
                    dma.advance(a);
                    dma.load(at_lds + NEXT * 2 * TB, at_lds + NEXT * 2 * TB + TB);
                    if (son) word_to_lds(sp + r0 + BR, lane * 4, at_stat + NEXT * (unsigned)sizeof(stat[0]));
                }
                step(std::false_type{}, NOW, r0);
                r0 += BR;
            };
            // Two steps at a time: the buffers' places are part of the instructions (heads of 128, 5 prompts of 601 .. 5184: 1339 -> 1280 us; the forward and gq gain nothing)
            int t = 0;
            for (; t + 1 < nfull; t += 2) {
                full(std::integral_constant<int, 0>{}, t);
                full(std::integral_constant<int, 1>{}, t + 1);
            }
            if (t < nfull) full(std::integral_constant<int, 0>{}, t);
        }
        if (r0 < R) border(r0);
        if (live) {
            T *ok = gk + ((sk.begin + key) * a.Hk + kv) * a.D, *ov = gv + ((sk.begin + key) * a.Hk + kv) * a.D;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                store_cols(ok, st.ak[d], d, h, a.D, a.scale);
                store_cols(ov, st.av[d], d, h, a.D, 1.f);
            }
            if (__builtin_expect(odd[wave], 0)) {
                int again = k0;
                asm volatile("" : "+s"(again));         // (all worked out again: kept, it would take registers from the loop)
                const int head = first_row(again), full = head + (max(first_row(min(again + BK, sk.n) - 1) - head, 0) + BR - 1) / BR * BR;
                const int tail = full < R ? R - (R - full) % BR : R;
                const long long at = sk.begin + again + wave * 32 + (lane & 31);
                const T *kr = (const T*)a.k + at * a.k_st + kv * a.k_sh, *vr = (const T*)a.v + at * a.v_st + kv * a.v_sh;
#pragma unroll 1
                for (int part = 0; part < 2; ++part)
                    add_spoilt(ok, ov, a, qrows, grows, kr, vr, rowstat, all, part ? max(tail, first_row(key)) : first_row(key), part ? R : min(full, R), h);
            }
        }
    }
}

// -------------------------------------------------------------- the backward where its tiles of 128 would leave the chip idle
// Tiles of 32 rows (gq) or keys (gk, gv); a workgroup's NW waves take the blocks of 32 of the other side in turn, with tiles of their own
// and no barrier, and their results meet in LDS in a fixed order.  NW = 1 where there is not more than one block or two.
template <typename T, int DP, int NW>
struct SplitCfg {
    static constexpr int TB = 32 * DP * (int)sizeof(T), LDS = NW * 4 * TB;
    static constexpr int WAVES = LDS / NW >= 32768 || LDS > 65536 ? 1 : LDS / NW <= 8192 ? 3 : 2;       // per SIMD
};

// NW results of 32 rows x DP (lane: row) summed over the waves: each thread gets four neighbouring columns of a row
template <typename T, int DP, int NW, typename F>
__device__ __forceinline__ void over_waves(float* pool, const f32x16* acc, int lane, int wave, int D, F out) {
    const int h = lane >> 5;
    __syncthreads();
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4*>(pool + (wave * 32 + (lane & 31)) * DP + ((d * 32 + 8 * g + 4 * h) ^ ((lane & 7) << 2))) =
                make_float4(acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]);
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * (DP / 4); i += NW * 64) {
        const int r = i / (DP / 4), d = (i % (DP / 4)) * 4;
        if (d >= D) continue;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(pool + (w * 32 + r) * DP + (d ^ ((r & 7) << 2)));
            o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
        }
        out(r, d, o);
    }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float4& o, float mul) {
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(p) = make_uint2(pack2(o.x * mul, o.y * mul), pack2(o.z * mul, o.w * mul));
    else *reinterpret_cast<float4*>(p) = make_float4(o.x * mul, o.y * mul, o.z * mul, o.w * mul);
}

template <typename T, int DP, int NW>
__global__ __launch_bounds__((NW * 64), (SplitCfg<T, DP, NW>::WAVES)) void k_attn_gq_split(Attn a, int tiles, unsigned first_rest) {
    constexpr int KS = DP / 16, DT = DP / 32, TB = SplitCfg<T, DP, NW>::TB;
    __shared__ __attribute__((aligned(1024))) char lds[SplitCfg<T, DP, NW>::LDS];
    __shared__ float part[NW][32], mul[32];
    __shared__ int odd;             // a key at the border was not finite
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    T* gq = (T*)a.gq;
    if (blockIdx.x >= first_rest) {
        const Rest z = rest(a.cu_q, a.B, a.Tq);
        for (long long i = (long long)(blockIdx.x - first_rest) * (NW * 8) + (threadIdx.x >> 3); i < z.n * a.Hq; i += (long long)(gridDim.x - first_rest) * (NW * 8))
            zero_row(gq + (z.row(i / a.Hq) * a.Hq + i % a.Hq) * a.D, a.D, threadIdx.x & 7, 8);
        return;
    }
    const Place pl = place(blockIdx.x, a.B * a.Hk, tiles);
    if (pl.tile < 0) return;
    const int b = pl.pair / a.Hk, kv = pl.pair - b * a.Hk;
    const Span sq = span(a.cu_q, nullptr, b, a.Tq), sk = span(a.cu_k, nullptr, b, a.Tk);
    const int R = sq.n * a.G;
    if ((long long)pl.tile * 32 >= R) return;
    const Rows qrows{sq.begin, a.q_st, a.q_sh, a.G, kv * a.G}, grows{sq.begin, a.go_st, a.go_sh, a.G, kv * a.G};
    const T *k = (const T*)a.k + sk.begin * a.k_st + kv * a.k_sh, *v = (const T*)a.v + sk.begin * a.v_st + kv * a.v_sh;
    const float c2 = a.scale * LOG2E;
    char* mine = lds + wave * 4 * TB;
    const unsigned at_lds = lds_at(mine);
    const Dma<T, DP, 32, 64> dk(a.k_st, a.D), dv(a.v_st, a.D);
    for (long long rr = (long long)pl.tile * 32; rr < R; rr += (long long)tiles * 32) {
        const int r0 = (int)rr, row = r0 + (lane & 31);
        const bool live = row < R;
        const int tok = live ? row / a.G : 0;
        const long long at = live ? (sq.begin + tok) * a.Hq + kv * a.G + (row - tok * a.G) : 0;
        const int jmax = live ? seen_keys(tok, sq.n, sk.n, a.causal) : 0;
        const int jend = seen_keys((min(r0 + 32, R) - 1) / a.G, sq.n, sk.n, a.causal), jall = seen_keys(r0 / a.G, sq.n, sk.n, a.causal);
        __syncthreads();
        if (a.D < DP)
            for (int i = lane; i < 4 * TB / 16; i += 64) reinterpret_cast<uint4*>(mine)[i] = make_uint4(0, 0, 0, 0);
        if (threadIdx.x == 0) odd = 0;
        __syncthreads();
        GqState<T, DP, 32> st;
        const float2 stat = live ? a.stats[at] : make_float2(0.f, 0.f);
        st.base = stat.x;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = s * 16 + h * 8;
            const bool on = live && d < a.D;
            st.qf[s] = frag_global((const T*)a.q + (live ? qrows.at(row) : 0) + d, on);
            st.gf[s] = frag_global((const T*)a.go + (live ? grows.at(row) : 0) + d, on);
        }
        // a block with a mask, through registers; checked: whether there is a key in it that is not finite
        const auto bring = [&](auto checked, int k0) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            const bool bad = stage<T, DP, 32, decltype(checked)::value, 64>(mine, k + (long long)k0 * a.k_st, sk.n - k0, a.D, [&](int r) { return (long long)r * a.k_st; });
            stage<T, DP, 32, false, 64>(mine + TB, v + (long long)k0 * a.v_st, sk.n - k0, a.D, [&](int r) { return (long long)r * a.v_st; });
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            return __any(bad);
        };
        float delta = 0.f;
        if (jend <= EXACT_D) {
            st.delta = st.sum = 0.f;
            for (int k0 = wave * 32; k0 < jend; k0 += NW * 32) {
                bring(std::false_type{}, k0);
                st.template step<true, true>(mine, mine + TB, lane, c2, jmax - k0);
            }
            delta = st.sum + __shfl_xor(st.sum, 32, 64);
            if (h == 0) part[wave][lane & 31] = delta;
            __syncthreads();
            delta = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) delta += part[w][lane & 31];
            delta *= stat.y;
        } else {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = s * 16 + h * 8;
                if (live && d < a.D) {
                    Raw8<T> x, y;
                    float fx[8], fy[8];
                    x.load((const T*)a.o + at * a.D + d);
                    y.load((const T*)a.go + grows.at(row) + d);
                    x.get(fx);
                    y.get(fy);
#pragma unroll
                    for (int j = 0; j < 8; ++j) delta += fx[j] * fy[j];
                }
            }
            delta += __shfl_xor(delta, 32, 64);
        }
        st.delta = delta;
        if (wave == 0 && live && h == 0) {
            const long long all = a.Tq * a.Hq;
            float* to = a.rowstat + ((long long)kv * a.Tq + sq.begin) * a.G + row;
            to[0] = sizeof(T) == 4 ? stat.x : stat.x - __builtin_amdgcn_logf(stat.y);
            to[all] = delta;
            if (sizeof(T) == 4) to[2 * all] = stat.y;
        }
#pragma unroll
        for (int i = 0; i < DT; ++i) st.acc[i] = zero16();
        const int full = jall / 32;
        int blk = wave, buf = 0;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (blk < full) {
            dk.load(k + (long long)blk * 32 * a.k_st, a.k_st, at_lds);
            dv.load(v + (long long)blk * 32 * a.v_st, a.v_st, at_lds + TB);
            wait_loads<0>();
        }
        for (; blk < full; blk += NW, buf ^= 1) {
            char* now = mine + buf * 2 * TB;
            const unsigned next = at_lds + (buf ^ 1) * 2 * TB;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (blk + NW < full) {
                dk.load(k + (long long)(blk + NW) * 32 * a.k_st, a.k_st, next);
                dv.load(v + (long long)(blk + NW) * 32 * a.v_st, a.v_st, next + TB);
                wait_loads<2 * Dma<T, DP, 32, 64>::N>();
            } else {
                wait_loads<0>();
            }
            st.template step<false, false, true>(now, now + TB, lane, c2, 32);
        }
        for (; blk * 32 < jend; blk += NW) {
            if (bring(std::true_type{}, blk * 32)) {
                odd = 1;
                clear_spoilt<T, DP, 64>(mine, k + (long long)blk * 32 * a.k_st, a.k_st, min(sk.n - blk * 32, 32), a.D);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
            st.template step<true, false, true>(mine, mine + TB, lane, c2, jmax - blk * 32);
        }
        if (wave == 0 && h == 0) mul[lane & 31] = a.scale * stat.y;
        over_waves<T, DP, NW>(reinterpret_cast<float*>(lds), st.acc, lane, wave, a.D, [&](int r, int d, const float4& o) {
            if (r0 + r >= R) return;
            const int t = (r0 + r) / a.G;
            store4(gq + ((sq.begin + t) * a.Hq + kv * a.G + (r0 + r - t * a.G)) * a.D + d, o, mul[r]);
        });
        if (odd) {          // (read behind the barriers of over_waves)
            __syncthreads();
            if (wave == 0 && live)
                st.add_spoilt(gq + at * a.D, a.scale * stat.y, (const T*)a.q + qrows.at(row), (const T*)a.go + grows.at(row), k, a.k_st, v, a.v_st, full * 32, jmax, a.D, h, c2);
        }
    }
}

template <typename T, int DP, int NW, bool EVEN>
__global__ __launch_bounds__((NW * 64), (SplitCfg<T, DP, NW>::WAVES)) void k_attn_gkv_split(Attn a, int tiles, unsigned first_rest) {
    constexpr int TB = SplitCfg<T, DP, NW>::TB;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int NS = F32 ? 3 : 2;
    __shared__ __attribute__((aligned(1024))) char lds[SplitCfg<T, DP, NW>::LDS];
    __shared__ __attribute__((aligned(1024))) float stat[NW][2][NS][32];
    __shared__ int odd;             // a row at the border was not finite
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    T *gk = (T*)a.gk, *gv = (T*)a.gv;
    if (blockIdx.x >= first_rest) {
        const Rest z = rest(a.cu_k, a.B, a.Tk);
        for (long long i = (long long)(blockIdx.x - first_rest) * (NW * 8) + (threadIdx.x >> 3); i < z.n * a.Hk; i += (long long)(gridDim.x - first_rest) * (NW * 8)) {
            const long long r = z.row(i / a.Hk) * a.Hk + i % a.Hk;
            zero_row(gk + r * a.D, a.D, threadIdx.x & 7, 8);
            zero_row(gv + r * a.D, a.D, threadIdx.x & 7, 8);
        }
        return;
    }
    const Place pl = place(blockIdx.x, a.B * a.Hk, tiles);
    if (pl.tile < 0) return;
    const int tile = tiles - 1 - pl.tile;
    const int b = pl.pair / a.Hk, kv = pl.pair - b * a.Hk;
    const Span sq = span(a.cu_q, nullptr, b, a.Tq), sk = span(a.cu_k, nullptr, b, a.Tk);
    if ((long long)tile * 32 >= sk.n) return;
    const int R = sq.n * a.G;
    const Rows qrows{sq.begin, a.q_st, a.q_sh, a.G, kv * a.G}, grows{sq.begin, a.go_st, a.go_sh, a.G, kv * a.G};
    const T *k = (const T*)a.k + sk.begin * a.k_st + kv * a.k_sh, *v = (const T*)a.v + sk.begin * a.v_st + kv * a.v_sh;
    const T *q0 = (const T*)a.q + sq.begin * a.q_st + (long long)kv * a.G * a.q_sh, *g0 = (const T*)a.go + sq.begin * a.go_st + (long long)kv * a.G * a.go_sh;
    const float c2 = a.scale * LOG2E;
    const long long all = a.Tq * a.Hq;
    char* mine = lds + wave * 4 * TB;
    const unsigned at_lds = lds_at(mine), at_stat = lds_at(&stat[wave][0][0][0]);
    const float* rowstat = a.rowstat + ((long long)kv * a.Tq + sq.begin) * a.G;
    for (long long kk = (long long)tile * 32; kk < sk.n; kk += (long long)tiles * 32) {
        const int k0 = (int)kk, key = k0 + (lane & 31);
        const bool live = key < sk.n;
        __syncthreads();
        if (a.D < DP)
            for (int i = lane; i < 4 * TB / 16; i += 64) reinterpret_cast<uint4*>(mine)[i] = make_uint4(0, 0, 0, 0);
        if (threadIdx.x == 0) odd = 0;
        __syncthreads();
        GkvState<T, DP, false> st;
        st.begin(k + (live ? key * a.k_st : 0), v + (live ? key * a.v_st : 0), live, a.D, h);
        const auto first_row = [&](int j) {
            const long long t = a.causal ? (long long)j - (sk.n - sq.n) : 0;
            return (t < 0 ? 0 : t > sq.n ? sq.n : (int)t) * a.G;
        };
        const int first = first_row(k0), r_all = first_row(min(k0 + 32, sk.n) - 1), r_key = live ? first_row(key) : R;
        // steps of 32 rows from `first`: those below `lo` and the last one, if it is short, need a mask.  One wave takes all of them that way: it
        // has two at most, and with FINE an infinity in go that a weight's rest multiplies would come out as NaN
        const int steps = R > first ? (R - first + 31) / 32 : 0, lo = NW == 1 ? steps : min((r_all - first + 31) / 32, steps), hi = max(lo, R > first ? (R - first) / 32 : 0);
        const auto border = [&](int s) {
            const int r0 = first + s * 32;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (lane < 32) {
                const bool on = r0 + lane < R;
#pragma unroll
                for (int i = 0; i < NS; ++i) stat[wave][0][i][lane] = on ? rowstat[i * all + r0 + lane] : 0.f;
            }
            bool bad = stage<T, DP, 32, true, 64>(mine, (const T*)a.q, R - r0, a.D, [&](int r) { return qrows.at(r0 + r); });
            bad |= stage<T, DP, 32, true, 64>(mine + TB, (const T*)a.go, R - r0, a.D, [&](int r) { return grows.at(r0 + r); });
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            st.template step<true, NW == 1>(mine, mine + TB, nullptr, &stat[wave][0][0][0], 32, lane, c2, r0, r_key, R);
            if (__any(bad)) odd = 1;
        };
        int s = wave;
        for (; s < lo; s += NW) border(s);
        if (NW > 1 && s < hi) {
            RowDma<T, DP, 32, EVEN, 64, NW * 32> dma(q0, g0, a, first + s * 32);
            const auto load = [&](unsigned to, unsigned st_to, int r0) {
                dma.load(to, to + TB);
#pragma unroll
                for (int i = 0; i < NS; ++i)
                    if (lane < 32) word_to_lds(rowstat + i * all + r0, lane * 4, st_to + i * 128);
            };
            constexpr int LOADS = 2 * RowDma<T, DP, 32, EVEN, 64, NW * 32>::N + NS;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            load(at_lds, at_stat, first + s * 32);
            wait_loads<0>();
            for (int buf = 0; s < hi; s += NW, buf ^= 1) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (s + NW < hi) {
                    dma.advance(a);
                    load(at_lds + (buf ^ 1) * 2 * TB, at_stat + (buf ^ 1) * NS * 128, first + (s + NW) * 32);
                    wait_loads<LOADS>();
                } else {
                    wait_loads<0>();
                }
                char* now = mine + buf * 2 * TB;
                st.template step<false, NW == 1>(now, now + TB, nullptr, &stat[wave][buf][0][0], 32, lane, c2, first + s * 32, r_key, R);
            }
        }
        for (; s < steps; s += NW) border(s);
        float* pool = reinterpret_cast<float*>(lds);
        over_waves<T, DP, NW>(pool, st.ak, lane, wave, a.D, [&](int r, int d, const float4& o) {
            if (k0 + r < sk.n) store4(gk + ((sk.begin + k0 + r) * a.Hk + kv) * a.D + d, o, a.scale);
        });
        over_waves<T, DP, NW>(pool, st.av, lane, wave, a.D, [&](int r, int d, const float4& o) {
            if (k0 + r < sk.n) store4(gv + ((sk.begin + k0 + r) * a.Hk + kv) * a.D + d, o, 1.f);
        });
        if (odd) {          // (read behind the barriers of over_waves)
            __syncthreads();
            if (wave == 0 && live) {
                T *ok = gk + ((sk.begin + key) * a.Hk + kv) * a.D, *ov = gv + ((sk.begin + key) * a.Hk + kv) * a.D;
                add_spoilt(ok, ov, a, qrows, grows, k + key * a.k_st, v + key * a.v_st, rowstat, all, r_key, min(first + lo * 32, R), h);
                add_spoilt(ok, ov, a, qrows, grows, k + key * a.k_st, v + key * a.v_st, rowstat, all, max(first + hi * 32, r_key), R, h);
            }
        }
    }
}

bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }
bool bad_pitch(int64_t ld, int dtype) { return (ld % (dtype == 0 ? 8 : 4)) != 0; }

int check(int64_t Tq, int64_t Tk, int B, int Hq, int Hk, int D, int64_t max_q, int64_t max_k, float scale, int dtype) {
    if (dtype != 0 && dtype != 1) return sam3_seq_fail(EINVAL_, "dtype must be 0 (bf16) or 1 (fp32), got %d", dtype);
    if (Tq < 0 || Tk < 0 || B < 0 || Hq <= 0 || Hk <= 0 || D <= 0 || max_q < 0 || max_k < 0) return sam3_seq_fail(EINVAL_, "attention: bad sizes");
    if (Hq % Hk) return sam3_seq_fail(EINVAL_, "attention: %d query heads over %d key heads", Hq, Hk);
    if (D % 8) return sam3_seq_fail(EINVAL_, "attention: head size must be a multiple of 8, got %d", D);
    if (D > 128) return sam3_seq_fail(ENOTSUP_, "attention: head size at most 128, got %d", D);
    if ((int64_t)B * Hk > 0x7ffffff) return sam3_seq_fail(ENOTSUP_, "attention: too many sequences and heads");
    if (B > 65000 || Hk > 65000) return sam3_seq_fail(ENOTSUP_, "attention: at most 65000 sequences and key heads");
    if (Tq * Hq > 0x7fff0000ll || Tk > 0x7fff0000ll) return sam3_seq_fail(ENOTSUP_, "attention: too many rows");
    if (!(scale > 0.f) || scale > 3.0e38f) return sam3_seq_fail(EINVAL_, "attention: scale must be positive and finite");
    return 0;
}
// Offsets inside a tile of 64 rows are 32 bits: between tokens, and where a tile's rows are a group's heads (grouped) between these.  Key
// heads are chosen by workgroups, in 64 bits: a cache may have its heads outside.
int check_tensor(const char* name, const void* p, int64_t st, int64_t sh, bool grouped, int dtype) {
    if (!p) return sam3_seq_fail(EINVAL_, "attention: %s is a null pointer", name);
    if (misaligned(p) || bad_pitch(st, dtype) || bad_pitch(sh, dtype))
        return sam3_seq_fail(EINVAL_, "attention: %s: pointer and strides must keep 16-byte accesses aligned", name);
    if (st < 0 || sh < 0) return sam3_seq_fail(EINVAL_, "attention: %s: negative strides", name);
    if (st >= (1 << 22) || (grouped && sh >= (1 << 22)))
        return sam3_seq_fail(ENOTSUP_, "attention: %s: rows must be less than 2^22 elements apart", name);
    return 0;
}

constexpr unsigned REST = 32;       // workgroups that clear the rows of no sequence (mostly there are none)

#define BY_HEAD(KERNEL, FLAG, GRID, ST, ...)                                                                         \
    do {                                                                                                        \
        if (dtype == 0) {                                                                                       \
            if (D <= 32) hipLaunchKernelGGL((KERNEL<bf16_t, 32, FLAG>), GRID, dim3(256), 0, ST, __VA_ARGS__);                 \
            else if (D <= 64) hipLaunchKernelGGL((KERNEL<bf16_t, 64, FLAG>), GRID, dim3(256), 0, ST, __VA_ARGS__);            \
            else hipLaunchKernelGGL((KERNEL<bf16_t, 128, FLAG>), GRID, dim3(256), 0, ST, __VA_ARGS__);                        \
        } else {                                                                                                \
            if (D <= 32) hipLaunchKernelGGL((KERNEL<float, 32, FLAG>), GRID, dim3(256), 0, ST, __VA_ARGS__);                  \
            else if (D <= 64) hipLaunchKernelGGL((KERNEL<float, 64, FLAG>), GRID, dim3(256), 0, ST, __VA_ARGS__);             \
            else hipLaunchKernelGGL((KERNEL<float, 128, FLAG>), GRID, dim3(256), 0, ST, __VA_ARGS__);                         \
        }                                                                                                       \
    } while (0)

unsigned tiles(int64_t rows, int per) {
    const int64_t t = (rows + per - 1) / per;
    return (unsigned)(t < 1 ? 1 : t);
}

// The tiles for each pair and the places of a launch; listed: one tile for a workgroup.  A grid has fewer than 2^32 threads.
struct Grid {
    int tiles;
    long long places;
    int threads;            // of a workgroup
    bool listed = false;
    bool fits() const { return (places + REST) * threads < 1ll << 32; }
    unsigned first_rest() const { return (unsigned)places; }
    dim3 grid() const { return dim3((unsigned)(places + REST)); }
};
// Tiles of `per` rows for each pair of a sequence and a key head: as many as the longest has, or listed (`total` rows lie in all) where that is
// over four times what there can be.  Measured on both sides (us, the longest's / listed; heads of 128, 32 / 8; forward, then backward):
// sequences of 1 .. 2048, 1.8 times: 707 / 692, 2576 / 2863; 64 of 512 and one of 4096, 6.8 times: 682 / 572, 2264 / 2346; 255 of 256 and one of
// 4096, 13 times: 1305 / 884, 4796 / 3514; 400 of 150 without hints, 216 times (16 heads of 64): 3958 / 309, 8633 / 849.
Grid tiled(int64_t longest, int64_t total, int B, int Hk, int per) {
    const int64_t all = Hk * (total / per + B);
    const int each = (int)tiles(longest, per);
    return places(B * Hk, each) > 4 * all + 4096 ? Grid{1 << 25, all, 256, true} : Grid{each, places(B * Hk, each), 256};
}

// The forward for few rows: rows of one token's heads or so (96 prompts of 2 .. 32 tokens: 19 us in tiles of 128, 11 in tiles of 32), or
// where the tiles of 128 rows would leave most of the chip idle and there are keys to split.  In tiles of 128 / split and joined (us, heads of
// 128): 16 tiles over 1024 keys 33 / 31, 64 over 8192 200 / 160, 128 over 8192 206 / 292, 128 over 4096 109 / 161.
struct Plan {
    bool few;
    int tiles, splits, chunk;
};
Plan plan(int64_t Tq, int B, int Hq, int Hk, int64_t max_q, int64_t max_k) {
    const int64_t rows = (max_q < Tq ? max_q : Tq) * (Hq / Hk), pairs = (int64_t)B * Hk;
    Plan p{};
    p.few = rows <= 32 || (max_k >= 256 && max_k >= 4 * max_q && pairs * tiles(rows, BM) <= 64);
    if (!p.few) return p;
    p.tiles = (int)tiles(rows, 32);
    // Chunks of 256 to 1024 keys as long as that gives 1024 waves, four for each CU; longer ones for a lot of keys, where 8192 of them
    // even out different lengths (24 requests of 1 .. 32768 keys, three draws: 437, 376 and 366 us; 4096 chunks 403, 386 and 383; 2048 486, 464
    // and 442).
    const int64_t keys = max_k * pairs * p.tiles;
    int64_t chunk = keys / 1024 < 1024 ? keys / 1024 : 1024;
    if (chunk < 256) chunk = 256;
    if (chunk < keys / 8192) chunk = keys / 8192;
    // The chunks' results take room for every row of q there is, sequence or not: no more of them than 2 GiB hold (8192 waves of 32 rows have 136 MB)
    const int64_t fit = (1ll << 31) / (Tq * Hq * (128 * 4 + 8) + 1), most = fit > 1 ? fit : 1;
    if (chunk * most < max_k) chunk = (max_k + most - 1) / most;
    chunk = (chunk + 127) / 128 * 128;
    p.chunk = (int)(chunk > 0x40000000 ? 0x40000000 : chunk);
    p.splits = (int)((max_k + p.chunk - 1) / p.chunk);
    if (p.splits < 1) p.splits = 1;
    return p;
}
// The backward's launches.  Tiles of 32, shared by the waves of a workgroup, where tiles of 128 would be too few for the chip.  Measured on both
// sides (us, tiles of 128 / of 32; causal sequences of 2048, one query head to a key head, tiles of 128 counted):
//   gq      bf16, heads of 128   128: 76 / 52, 256: 82 / 103;    of 64   128: 39 / 25, 256: 41 / 39, 512: 56 / 75
//           fp32, heads of 64    128: 221 / 90, 256: 227 / 174, 384: 402 / 256, 1024: 660 / 674;    of 128   64: 421 / 415, 128: 424 / 498
//   gk, gv  bf16, heads of 128   128: 107 / 53, 256: 118 / 104, 384: 140 / 153;    of 64   256: 55 / 38, 384: 68 / 59, 512: 70 / 73
//           fp32, heads of 64    256: 289 / 205, 512: 508 / 407, 1024: 842 / 808;    of 128   64: 521 / 433, 128: 526 / 491, 256: 530 / 969
// Sequences of 512 change sides earlier (gk, gv of heads of 128: bf16 at 192, 50 / 56; fp32 at 64, 148 / 141).
struct Backward {
    bool q_split, k_split;
    Grid q, k;
};
Backward backward_of(int64_t Tq, int64_t Tk, int B, int G, int Hk, int D, int64_t longest_q, int64_t longest_k, int dtype) {
    const int64_t pairs = (int64_t)B * Hk, rows = longest_q * G;
    Backward b;
    const bool wide = dtype == 1 && D > 64;         // (two waves of 512 registers each share a tile then)
    b.q_split = pairs * tiles(rows, BM) <= (wide ? 64 : 128) || rows <= 32;
    b.k_split = pairs * tiles(longest_k, 128) <= (wide ? 96 : 256) || longest_k <= 32;
    const int qt = (int)tiles(rows, 32), kt = (int)tiles(longest_k, 32);
    b.q = b.q_split ? Grid{qt, places(B * Hk, qt), 256} : tiled(rows, Tq * G, B, Hk, BM);
    b.k = b.k_split ? Grid{kt, places(B * Hk, kt), 256} : tiled(longest_k, Tk, B, Hk, 128);
    return b;
}
size_t part_bytes(int64_t Tq, int Hq, int D, int splits) {
    return splits > 1 ? (size_t)splits * Tq * Hq * (D * sizeof(float) + sizeof(float2)) : 0;
}

}  // namespace

extern "C" {

size_t sam3_seq_attn_fwd_workspace_bytes(int64_t Tq, int B, int Hq, int Hk, int D, int64_t max_q, int64_t max_k, int dtype) {
    if (check(Tq, 0, B, Hq, Hk, D, max_q, max_k, 1.f, dtype) || Tq == 0) return 0;
    const Plan p = plan(Tq, B, Hq, Hk, max_q, max_k);
    return p.few ? part_bytes(Tq, Hq, D, p.splits) : 0;
}

int sam3_seq_attn_fwd(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                      int64_t v_st, int64_t v_sh, const int32_t* cu_q, const int32_t* cu_k, const int32_t* len_k, void* out,
                      float* lse, float* stats, int64_t Tq, int64_t Tk, int B, int Hq, int Hk, int D, int64_t max_q, int64_t max_k, int causal,
                      float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    sam3_seq_clear_error();
    if (int rc = check(Tq, Tk, B, Hq, Hk, D, max_q, max_k, scale, dtype)) return rc;
    if (Tq == 0) return 0;
    if (int rc = check_tensor("q", q, q_st, q_sh, Hq > Hk, dtype)) return rc;
    if (Tk > 0) {
        if (int rc = check_tensor("k", k, k_st, k_sh, false, dtype)) return rc;
        if (int rc = check_tensor("v", v, v_st, v_sh, false, dtype)) return rc;
    }
    if (!cu_q || !cu_k || !out || misaligned(out)) return sam3_seq_fail(EINVAL_, "attention: null or misaligned pointer");
    if (B == 0) max_q = max_k = 0;
    Attn a{};
    a.q = q; a.k = k; a.v = v; a.out = out; a.lse = lse; a.stats = (float2*)stats; a.cu_q = cu_q; a.cu_k = cu_k; a.len_k = len_k;
    a.q_st = q_st; a.q_sh = q_sh; a.k_st = k_st; a.k_sh = k_sh; a.v_st = v_st; a.v_sh = v_sh;
    a.Tq = Tq; a.Tk = Tk; a.B = B; a.Hq = Hq; a.Hk = Hk; a.G = Hq / Hk; a.D = D; a.causal = causal; a.scale = scale;
    const Plan p = plan(Tq, B, Hq, Hk, max_q, max_k);
    if (p.few) {
        const size_t need = part_bytes(Tq, Hq, D, p.splits);
        if (need && (!workspace || workspace_bytes < need || misaligned(workspace)))
            return sam3_seq_fail(ENOMEM_, "attention: workspace too small or misaligned: %zu < %zu", workspace_bytes, need);
        const long long items = (long long)B * Hk * p.splits;
        if (items > 0x3fffffffll) return sam3_seq_fail(ENOTSUP_, "attention: too many tiles of rows");
        const Grid g{p.tiles, places((int)items, p.tiles), 64};
        if (!g.fits()) return sam3_seq_fail(ENOTSUP_, "attention: too many tiles of rows");
        Few f{p.tiles, p.splits, p.chunk, (float*)workspace, nullptr, g.first_rest()};
        f.pstat = reinterpret_cast<float2*>(f.part + (p.splits > 1 ? (size_t)p.splits * Tq * Hq * D : 0));
        const dim3 grid = g.grid();
        hipStream_t st = (hipStream_t)stream;
#define FEW(TY, W)                                                                                                    \
    do {                                                                                                              \
        if (sizeof(TY) == 2 && p.tiles == 1) hipLaunchKernelGGL((k_attn_few<TY, W, sizeof(TY) == 2>), grid, dim3(64), 0, st, a, f); \
        else hipLaunchKernelGGL((k_attn_few<TY, W, false>), grid, dim3(64), 0, st, a, f);                             \
    } while (0)
        if (dtype == 0) { if (D <= 32) FEW(bf16_t, 32); else if (D <= 64) FEW(bf16_t, 64); else FEW(bf16_t, 128); }
        else { if (D <= 32) FEW(float, 32); else if (D <= 64) FEW(float, 64); else FEW(float, 128); }
#undef FEW
        if (int rc = launched("sam3_seq_attn_fwd")) return rc;
        if (p.splits > 1 && B > 0) {
            const int64_t rows = (max_q < Tq ? max_q : Tq) * Hq;
            const dim3 jgrid(tiles(rows, 1) < 8192 ? tiles(rows, 1) : 8192, (unsigned)B);
            if (dtype == 0) hipLaunchKernelGGL(k_attn_join<bf16_t>, jgrid, dim3(256), 0, st, a, f);
            else hipLaunchKernelGGL(k_attn_join<float>, jgrid, dim3(256), 0, st, a, f);
        }
        return launched("sam3_seq_attn_fwd");
    }
    const Grid g = tiled((max_q < Tq ? max_q : Tq) * a.G, Tq * a.G, B, Hk, BM);
    if (!g.fits()) return sam3_seq_fail(ENOTSUP_, "attention: too many tiles of rows");
    if (g.listed) BY_HEAD(k_attn_fwd, true, g.grid(), (hipStream_t)stream, a, g.tiles, g.first_rest());
    else BY_HEAD(k_attn_fwd, false, g.grid(), (hipStream_t)stream, a, g.tiles, g.first_rest());
    return launched("sam3_seq_attn_fwd");
}

int64_t sam3_seq_attn_workgroups(int kernel, int64_t Tq, int64_t Tk, int B, int Hq, int Hk, int D, int64_t max_q, int64_t max_k, int dtype) {
    sam3_seq_clear_error();
    if (int rc = check(Tq, Tk, B, Hq, Hk, D, max_q, max_k, 1.f, dtype)) return rc;
    if (kernel < 0 || kernel > 2) return sam3_seq_fail(EINVAL_, "attention: no launch %d", kernel);
    if (B == 0) max_q = max_k = 0;
    const int64_t lq = max_q < Tq ? max_q : Tq, lk = max_k < Tk ? max_k : Tk;
    Grid g;
    if (kernel == 0) {
        const Plan p = plan(Tq, B, Hq, Hk, max_q, max_k);
        g = p.few ? Grid{p.tiles, places(B * Hk * p.splits, p.tiles), 64} : tiled(lq * (Hq / Hk), Tq * (Hq / Hk), B, Hk, BM);
    } else {
        const Backward w = backward_of(Tq, Tk, B, Hq / Hk, Hk, D, lq, lk, dtype);
        g = kernel == 1 ? w.q : w.k;
    }
    return g.fits() ? g.places + REST : sam3_seq_fail(ENOTSUP_, "attention: too many tiles of rows");
}

size_t sam3_seq_attn_bwd_workspace_bytes(int64_t Tq, int Hq) { return Tq > 0 && Hq > 0 ? (size_t)Tq * Hq * 3 * sizeof(float) : 0; }

int sam3_seq_attn_bwd(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                      int64_t v_st, int64_t v_sh, const void* go, int64_t go_st, int64_t go_sh, const void* out, const float* stats,
                      const int32_t* cu_q, const int32_t* cu_k, void* gq, void* gk, void* gv, int64_t Tq, int64_t Tk, int B, int Hq,
                      int Hk, int D, int64_t max_q, int64_t max_k, int causal, float scale, int dtype, void* workspace,
                      size_t workspace_bytes, void* stream) {
    sam3_seq_clear_error();
    if (int rc = check(Tq, Tk, B, Hq, Hk, D, max_q, max_k, scale, dtype)) return rc;
    if (Tq > 0) {
        if (int rc = check_tensor("q", q, q_st, q_sh, Hq > Hk, dtype)) return rc;
        if (int rc = check_tensor("go", go, go_st, go_sh, Hq > Hk, dtype)) return rc;
        if (!out || !stats || !gq || misaligned(out) || misaligned(gq)) return sam3_seq_fail(EINVAL_, "attention: null or misaligned pointer");
        if (!workspace || workspace_bytes < sam3_seq_attn_bwd_workspace_bytes(Tq, Hq))
            return sam3_seq_fail(ENOMEM_, "attention: workspace too small: %zu < %zu", workspace_bytes, sam3_seq_attn_bwd_workspace_bytes(Tq, Hq));
    }
    if (Tk > 0) {
        if (int rc = check_tensor("k", k, k_st, k_sh, false, dtype)) return rc;
        if (int rc = check_tensor("v", v, v_st, v_sh, false, dtype)) return rc;
        if (!gk != !gv || misaligned(gk) || misaligned(gv)) return sam3_seq_fail(EINVAL_, "attention: null or misaligned pointer");
    }
    if (!cu_q || !cu_k) return sam3_seq_fail(EINVAL_, "attention: null pointer");
    Attn a{};
    a.q = q; a.k = k; a.v = v; a.go = go; a.o = out; a.stats = (float2*)stats; a.rowstat = (float*)workspace;
    a.gq = gq; a.gk = gk; a.gv = gv; a.cu_q = cu_q; a.cu_k = cu_k;
    a.q_st = q_st; a.q_sh = q_sh; a.k_st = k_st; a.k_sh = k_sh; a.v_st = v_st; a.v_sh = v_sh; a.go_st = go_st; a.go_sh = go_sh;
    a.Tq = Tq; a.Tk = Tk; a.B = B; a.Hq = Hq; a.Hk = Hk; a.G = Hq / Hk; a.D = D; a.causal = causal; a.scale = scale;
    const int64_t longest_q = max_q < Tq ? max_q : Tq, longest_k = max_k < Tk ? max_k : Tk;
    const Backward w = backward_of(Tq, Tk, B, a.G, Hk, D, longest_q, longest_k, dtype);
    if (!w.q.fits() || (gk && !w.k.fits())) return sam3_seq_fail(ENOTSUP_, "attention: too many tiles of rows");
    const bool q_one = longest_k <= 64, k_one = longest_q * a.G <= 64;      // not more than two blocks for the waves to share
    hipStream_t st = (hipStream_t)stream;
    if (Tq > 0) {
        const dim3 grid = w.q.grid();
#define GQ(TY, W)                                                                                                                       \
    do {                                                                                                                                \
        constexpr int NW = sizeof(TY) * W > 256 ? 2 : 4;                                                                                \
        if (w.q.listed) hipLaunchKernelGGL((k_attn_gq<TY, W, true>), grid, dim3(256), 0, st, a, w.q.tiles, w.q.first_rest());             \
        else if (!w.q_split) hipLaunchKernelGGL((k_attn_gq<TY, W, false>), grid, dim3(256), 0, st, a, w.q.tiles, w.q.first_rest());                          \
        else if (q_one) hipLaunchKernelGGL((k_attn_gq_split<TY, W, 1>), grid, dim3(64), 0, st, a, w.q.tiles, w.q.first_rest());                \
        else hipLaunchKernelGGL((k_attn_gq_split<TY, W, NW>), grid, dim3(NW * 64), 0, st, a, w.q.tiles, w.q.first_rest());                     \
    } while (0)
        if (dtype == 0) { if (D <= 32) GQ(bf16_t, 32); else if (D <= 64) GQ(bf16_t, 64); else GQ(bf16_t, 128); }
        else { if (D <= 32) GQ(float, 32); else if (D <= 64) GQ(float, 64); else GQ(float, 128); }
#undef GQ
        if (int rc = launched("sam3_seq_attn_bwd")) return rc;
    }
    if (Tk > 0 && gk) {
        const dim3 grid = w.k.grid();
#define GKV(TY, W)                                                                                                                      \
    do {                                                                                                                                \
        constexpr int NW = sizeof(TY) * W > 256 ? 2 : 4;                                                                                \
        if (w.k.listed) hipLaunchKernelGGL((k_attn_gkv<TY, W, false, true>), grid, dim3(256), 0, st, a, w.k.tiles, w.k.first_rest());     \
        else if (!w.k_split) { if (GkvCfg<TY, W>::BR % a.G == 0) hipLaunchKernelGGL((k_attn_gkv<TY, W, true, false>), grid, dim3(256), 0, st, a, w.k.tiles, w.k.first_rest()); \
                        else hipLaunchKernelGGL((k_attn_gkv<TY, W, false, false>), grid, dim3(256), 0, st, a, w.k.tiles, w.k.first_rest()); }          \
        else if (k_one) { if (32 % a.G == 0) hipLaunchKernelGGL((k_attn_gkv_split<TY, W, 1, true>), grid, dim3(64), 0, st, a, w.k.tiles, w.k.first_rest());      \
                          else hipLaunchKernelGGL((k_attn_gkv_split<TY, W, 1, false>), grid, dim3(64), 0, st, a, w.k.tiles, w.k.first_rest()); } \
        else { if (32 % a.G == 0) hipLaunchKernelGGL((k_attn_gkv_split<TY, W, NW, true>), grid, dim3(NW * 64), 0, st, a, w.k.tiles, w.k.first_rest());           \
               else hipLaunchKernelGGL((k_attn_gkv_split<TY, W, NW, false>), grid, dim3(NW * 64), 0, st, a, w.k.tiles, w.k.first_rest()); }      \
    } while (0)
        if (dtype == 0) { if (D <= 32) GKV(bf16_t, 32); else if (D <= 64) GKV(bf16_t, 64); else GKV(bf16_t, 128); }
        else { if (D <= 32) GKV(float, 32); else if (D <= 64) GKV(float, 64); else GKV(float, 128); }
#undef GKV
    }
    return launched("sam3_seq_attn_bwd");
}

}  // extern "C"
