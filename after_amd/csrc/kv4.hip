// A key / value cache held in four bits, the attention that reads it, and the eviction of slots by the attention they received
// (include/after_hip.h: after_kv4_*; Python: after_amd.KVCache4).
//
// Format.  32 neighbouring channels of one token form a group: one byte b, the power of two 2^(b - 127), and 32 four-bit floats
// (sign, two bits of exponent, one of fraction: 0, .5, 1, 1.5, 2, 3, 4, 6).  17 bytes per 32 channels, against 64 of a 16-bit
// cache.  The power is the smallest with which the group's largest magnitude is <= 6, so nothing saturates (but beyond
// 6 * 2^125); gfx950 converts both ways in hardware (v_cvt_scalef32_pk_*_fp4, to nearest even).  Bytes run from 16 to 252:
// every value but 0 is a normal bf16 number, so that bf16 carries all of them exactly.  Byte 255 marks a group that held an
// infinity or NaN: it reads as NaN.
//
// Layout.  keys [rows][H][C][D / 2]: a token's channels side by side, two to a byte.  values [rows][H][C / 8][D][4]: eight
// tokens of a channel in a dword, since the product P V contracts over tokens: a lane's eight tokens of one channel are then one
// load and four conversions, and nothing is transposed on the way to the matrix pipe.  The channels of such a block stand in the
// order [d / 2 % 16][d / 32][d % 2]: what lane d / 2 % 16 of the product needs is one piece of D / 4 bytes.
#include <hip/hip_runtime.h>

#include <cmath>

#include "attention.h"
#include "common.h"
#include "gemm_pipe.h"

namespace after {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMinByte = 16, kMaxByte = 252, kBadByte = 255;

template <int TYPE>
struct Elem;
template <>
struct Elem<AFTER_T_F32> {
    using T = float;
};
template <>
struct Elem<AFTER_T_BF16> {
    using T = __bf16;
};
template <>
struct Elem<AFTER_T_F16> {
    using T = _Float16;
};

// N consecutive elements (N * sizeof(T) aligned) as floats
template <int N, typename T>
__device__ __forceinline__ void load_n(const T* p, float (&x)[N]) {
    typedef T vec __attribute__((ext_vector_type(N)));
    const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)v[i];
}
template <int N, typename T>
__device__ __forceinline__ void store_n(T* p, const float (&x)[N]) {
    typedef T vec __attribute__((ext_vector_type(N)));
    vec v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)x[i];
    *reinterpret_cast<vec*>(p) = v;
}

__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// the scale byte of a group whose largest magnitude has these bits: the smallest e with top <= 1.5 * 2^(e + 2)
__device__ __forceinline__ int scale_byte(unsigned top) {
    if (top >= 0x7F800000u) return kBadByte;
    const int b = (int)(top >> 23) - 2 + ((top & 0x7FFFFFu) > 0x400000u ? 1 : 0);
    return min(max(b, kMinByte), kMaxByte);
}
__device__ __forceinline__ float byte_scale(int b) { return __uint_as_float((unsigned)b << 23); }
__device__ __forceinline__ float scale_or_nan(unsigned b) { return __uint_as_float(b << 23 | (b + 1) >> 8); }  // (255: NaN)

// two floats -> the low byte: two codes
__device__ __forceinline__ unsigned round4(float a, float b, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, a, b, scale, 0) & 255u;
}
// the four bytes of a dword -> eight bf16 values (code * scale)
__device__ __forceinline__ bf16x8 widen8(unsigned w, float scale) {
    union {
        bf16x8 v;
        bf16x2 p[4];
    } u;
    u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0);
    u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
    u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2);
    u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
    return u.v;
}

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }
__device__ __forceinline__ int row_length(const after_kv4& c, int r) { return clampi(c.lengths[r], 0, c.capacity); }

// ---------------------------------------------------------------------------------------------------------------- append
struct NewTokens {
    const int* starts;  // [rows + 1], or nullptr: `each` tokens of every row
    int each;
    int total;
    __device__ __forceinline__ int start(int r) const { return starts ? clampi(starts[r], 0, total) : r * each; }
};

// the largest of 16 neighbouring lanes' values, in all of them (rotations inside the row: no LDS)
__device__ __forceinline__ unsigned row_max(unsigned x) {
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xF, 0xF, true));
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xF, 0xF, true));
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xF, 0xF, true));
    return max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xF, 0xF, true));
}
// ... of four
__device__ __forceinline__ unsigned quad_max(unsigned x) {
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, true));         // lanes 1 0 3 2
    return max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, true));  // lanes 2 3 0 1
}

// sums of the lanes up to this one (inside the vector unit: shuffles through LDS take several times as long)
__device__ __forceinline__ int lane_sums(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // 1, 2, 4, 8 lanes on, inside each 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // lane 15 of the 16 before to the second and fourth 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // lane 31 to the upper half
    return x;
}

struct AppendArgs {
    after_kv4 c;
    NewTokens nt;
    const void *k, *v;
    long long kts, khs, vts, vhs;
};

// One wave rounds those of a row's new tokens, len .. end, that fall into block sb of eight slots, for one head; t0: the row's first.
template <int TYPE, int D>
__device__ __forceinline__ void append_block(const AppendArgs& a, int r, int h, int t0, int len, int end, int sb) {
    using T = typename Elem<TYPE>::T;
    constexpr int G = D / 32;
    const after_kv4& c = a.c;
    const int lane = threadIdx.x & 63;
    const size_t rh = (size_t)r * c.kv_heads + h;
    const T* k = (const T*)a.k + (size_t)h * a.khs;
    const T* v = (const T*)a.v + (size_t)h * a.vhs;
    // keys: eight channels per lane; values: two channels of the eight tokens per lane.  Everything is asked for first.
    float x[D / 64][8], y[8][2];
    bool in[D / 64];
#pragma unroll
    for (int it = 0; it < D / 64; ++it) {
        const int id = it * 64 + lane, s = 8 * sb + id / (D / 8);
        in[it] = s >= len && s < end;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[it][i] = 0.f;
        if (in[it]) load_n<8, T>(k + (long long)(t0 + s - len) * a.kts + 8 * (id % (D / 8)), x[it]);
    }
    const bool holds = 2 * lane < D;
#pragma unroll
    for (int tt = 0; tt < 8; ++tt) {
        const int s = 8 * sb + tt;
        y[tt][0] = y[tt][1] = 0.f;
        if (holds && s >= len && s < end) load_n<2, T>(v + (long long)(t0 + s - len) * a.vts + 2 * lane, y[tt]);
    }
    if (lane < 8) {
        const int s = 8 * sb + lane;
        if (s >= len && s < end) c.weights[rh * c.capacity + s] = 0.f;
    }
#pragma unroll
    for (int it = 0; it < D / 64; ++it) {
        const int id = it * 64 + lane, ch = id % (D / 8), s = 8 * sb + id / (D / 8);
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, abs_bits(x[it][i]));
        const int b = scale_byte(quad_max(top));
        const float sc = byte_scale(b);
        unsigned w = round4(x[it][0], x[it][1], sc) | round4(x[it][2], x[it][3], sc) << 8 | round4(x[it][4], x[it][5], sc) << 16 | round4(x[it][6], x[it][7], sc) << 24;
        if (b == kBadByte) w = 0;
        if (in[it]) {
            *reinterpret_cast<unsigned*>(c.keys + (rh * c.capacity + s) * (D / 2) + 4 * ch) = w;
            if ((ch & 3) == 0) c.key_scales[(rh * c.capacity + s) * G + ch / 4] = (unsigned char)b;
        }
    }
    unsigned w0 = 0, w1 = 0, mask = 0;
    int mine = 0;  // lane tt of each 16: token tt's byte
#pragma unroll
    for (int tt = 0; tt < 8; ++tt) {
        const int s = 8 * sb + tt, b = scale_byte(row_max(max(abs_bits(y[tt][0]), abs_bits(y[tt][1]))));
        const unsigned u = b == kBadByte ? 0u : round4(y[tt][0], y[tt][1], byte_scale(b));
        w0 |= (u & 15u) << 4 * tt;
        w1 |= (u >> 4) << 4 * tt;
        mask |= s >= len && s < end ? 15u << 4 * tt : 0u;
        mine = (lane & 15) == tt ? b : mine;
    }
    if (holds) {
        const int s = 8 * sb + (lane & 15);
        if ((lane & 15) < 8 && s >= len && s < end) c.value_scales[(rh * c.capacity + s) * G + lane / 16] = (unsigned char)mine;
        u32x2* at = reinterpret_cast<u32x2*>(c.values + ((rh * (c.capacity / 8) + sb) * D + (lane & 15) * (D / 16) + (lane >> 4) * 2) * 4);
        u32x2 w = {w0 & mask, w1 & mask};
        if (mask != 0xFFFFFFFFu) {  // the other slots of the block keep what they hold
            const u32x2 old = *at;
            w = w | (old & ~mask);
        }
        *at = w;
    }
}

// A wave for each block and head.  Row r owns the block numbers from start(r) / 8 + 2 r on: at least as many as its tokens touch,
// wherever in a block they begin, so the grid needs no lengths.
template <int TYPE, int D>
__global__ __launch_bounds__(256) void kv4_append_kernel(AppendArgs a, int items) {
    const after_kv4& c = a.c;
    const int item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= items) return;
    const int h = item % c.kv_heads, fb = item / c.kv_heads, lane = threadIdx.x & 63;
    // the last row that begins at or before fb: 64 candidates at a time; the last look holds its tokens and length
    int lo = 0, hi = c.rows - 1, r, t0, n, len;
    for (;;) {
        const int step = (hi - lo + 64) >> 6, at = min(lo + lane * step, hi), t = a.nt.start(at), next = a.nt.start(at + 1), l = row_length(c, at);
        const int j = 63 - __clzll(__ballot(t / 8 + 2 * at <= fb && lo + lane * step <= hi) | 1);
        if (step == 1) {
            r = lo + j;
            t0 = __builtin_amdgcn_readlane(t, j);
            n = __builtin_amdgcn_readlane(next, j) - t0;
            len = __builtin_amdgcn_readlane(l, j);
            break;
        }
        lo += j * step;
        hi = min(hi, lo + step - 1);
    }
    const int sb = len / 8 + fb - (t0 / 8 + 2 * r), end = min(len + max(n, 0), c.capacity);  // tokens that do not fit are dropped
    if (sb >= 0 && 8 * sb < end) append_block<TYPE, D>(a, r, h, t0, len, end, sb);
}

__device__ __forceinline__ void advance(const after_kv4& c, const NewTokens& nt, int r, int len) {
    const int n = max(nt.start(r + 1) - nt.start(r), 0);
    if (n > c.capacity - len) *c.failed = 1;
    c.lengths[r] = min(n, c.capacity - len) + len;
}
__global__ void kv4_advance_kernel(after_kv4 c, NewTokens nt) {
    const int r = blockIdx.x * blockDim.x + threadIdx.x;
    if (r < c.rows) advance(c, nt, r, row_length(c, r));
}

// The same with a workgroup for each row, which also moves the row's length: one launch where there are few tokens.
template <int TYPE, int D>
__global__ __launch_bounds__(512) void kv4_append_rows_kernel(AppendArgs a) {
    const after_kv4& c = a.c;
    const int r = blockIdx.x, t0 = a.nt.start(r), n = a.nt.start(r + 1) - t0, len = row_length(c, r), end = min(len + max(n, 0), c.capacity);
    const int first = len / 8, blocks = end > len ? (end - 1) / 8 - first + 1 : 0;
    for (int i = threadIdx.x >> 6; i < blocks * c.kv_heads; i += 8) append_block<TYPE, D>(a, r, i % c.kv_heads, t0, len, end, first + i / c.kv_heads);
    __syncthreads();  // (every wave has read the length)
    if (threadIdx.x == 0) advance(c, a.nt, r, len);
}

__global__ void kv4_truncate_kernel(after_kv4 c, const int* lengths) {
    const int r = blockIdx.x * blockDim.x + threadIdx.x;
    if (r < c.rows) c.lengths[r] = lengths ? clampi(lengths[r], 0, row_length(c, r)) : 0;
}

// ---------------------------------------------------------------------------------------------------------------- read
// One wave per (row, head, block of eight slots): the slots [start, start + count) as values; past the row's length zeros.
template <int TYPE, int D>
__global__ __launch_bounds__(256) void kv4_read_kernel(after_kv4 c, void* ko, void* vo, const int* start, int count, int nb, long long items) {
    using T = typename Elem<TYPE>::T;
    constexpr int G = D / 32;
    const int lane = threadIdx.x & 63;
    const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (item >= items) return;
    const size_t rh = item / nb;
    const int r = (int)(rh / c.kv_heads);
    const int st = start ? clampi(start[r], 0, c.capacity) : 0;
    const int sb = st / 8 + (int)(item % nb);
    if (8 * sb >= st + count) return;
    const int len = row_length(c, r);
    T* k = (T*)ko + rh * count * D;
    T* v = (T*)vo + rh * count * D;
#pragma unroll
    for (int it = 0; it < D / 64; ++it) {
        const int id = it * 64 + lane, tt = id / (D / 8), ch = id % (D / 8), s = 8 * sb + tt, o = s - st;
        if (o < 0 || o >= count) continue;
        float x[8] = {};
        if (s < len) {
            const unsigned w = *reinterpret_cast<const unsigned*>(c.keys + (rh * c.capacity + s) * (D / 2) + 4 * ch);
            const bf16x8 y = widen8(w, byte_scale(c.key_scales[(rh * c.capacity + s) * G + ch / 4]));
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (float)y[i];
        }
        store_n<8, T>(k + (size_t)o * D + 8 * ch, x);
    }
    if (2 * lane < D) {
        u32x2 w = {0, 0};
        if (8 * sb < len) w = *reinterpret_cast<const u32x2*>(c.values + ((rh * (c.capacity / 8) + sb) * D + (lane & 15) * (D / 16) + (lane >> 4) * 2) * 4);
#pragma unroll
        for (int tt = 0; tt < 8; ++tt) {
            const int s = 8 * sb + tt, o = s - st;
            if (o < 0 || o >= count) continue;
            float x[2] = {};
            if (s < len) {
                const bf16x2 y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((w[0] >> 4 * tt & 15u) | (w[1] >> 4 * tt & 15u) << 4,
                                                                           byte_scale(c.value_scales[(rh * c.capacity + s) * G + lane / 16]), 0);
                x[0] = (float)y[0];
                x[1] = (float)y[1];
            }
            store_n<2, T>(v + (size_t)o * D + 2 * lane, x);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------- attend
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16: the 16 columns are (token, head of the group) pairs that share
// the cached head, the rows cached tokens / channels.  Everything stays in registers: which token a row of S^T stands for and
// which channel a step of its product contracts are chosen so that a lane's S values are the P operand that it needs next.
// A cached value is exact in bf16; queries and probabilities travel as bf16 pieces (1 for bf16 queries, 2 for fp16: exact,
// 3 for fp32: exact), so that what is rounded is never coarser than the output's own type.
// What bounds it: memory.  64 rows of 1 .. 8192 slots, 8 heads of 128 (296 MB): 57 us and 5.6 for the join, 5.2 TB/s (fp16 61, fp32
// 66); two rows of 131071 with 8 fp16 queries a head, whose scores are written for the weights (285 + 67 MB): 80 us, 4.4 TB/s: the
// stores of scores count in the counter that the ring waits on, so that its third tile is asked for late.  24 queries a head, 8 rows
// of 1 .. 32767: 57 us in bf16, 86 in fp16, 110 in fp32.
struct AttendArgs {
    after_kv4 c;
    const void* q;
    void* out;  // [rows][tokens][heads][D]
    long long qrs, qts, qhs;
    int heads, tokens, group, m_rows;  // m_rows = tokens * group
    int workers;      // waves that share the work (below); 0: a workgroup for each row and head
    int pieces;       // that part_o and part_ml hold
    float scale2;     // |scale| log2(e), > 0 (a masked score, -inf, stays -inf)
    float q_sign;     // the scale's sign, on the queries
    float* part_o;    // [pieces][m_rows][D]: a piece is one worker's part of a row and head, number worker + row * H + head (many
                      // queries: one workgroup's, number head * rows * splits + its place among the head's)
    f32x2* part_ml;   // [pieces][m_rows]: largest score, sum of exponentials to it
    f32x2* final_ml;  // [rows * H][m_rows]: the same over all pieces, if weights are wanted
    int2* ends;       // [rows * H]: the first and the last piece of a row and head, written by the workers that hold its ends
    float* scores;    // [rows * H][m_rows][C], not scaled, or nullptr
};

// How the slots in use are shared out: the steps of 32 slots of all rows and heads, one behind the other, are cut into equal
// shares, one for each wave on the chip, wherever that cuts a row.  So all end together however different the rows are, and
// there are no more ends than waves, rows and heads; no wave waits for another.  Lengths are on the device: every wave looks at
// them (64 at a time) before it begins.
constexpr int kStep = 32;
__device__ __forceinline__ long long wave_sum(long long x) {
#pragma unroll
    for (int o = 1; o < 64; o *= 2) x += __shfl_xor(x, o);
    return x;
}
__device__ __forceinline__ int row_steps(const after_kv4& c, int r) { return (row_length(c, r) + kStep - 1) / kStep; }
template <int N>
__device__ __forceinline__ void pieces8(const float (&x)[8], bf16x8 (&p)[N]) {
    float rest[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[n][i] = (__bf16)rest[i];
        if (n + 1 < N) {
#pragma unroll
            for (int i = 0; i < 8; ++i) rest[i] -= (float)p[n][i];
        }
    }
}

// ... of queries, exactly: all pieces but the last are cut off, not rounded, since fp32's largest numbers would become infinities
template <int N>
__device__ __forceinline__ void query_pieces8(const float (&x)[8], bf16x8 (&p)[N]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float rest = x[i];
#pragma unroll
        for (int n = 0; n < N - 1; ++n) {
            const unsigned u = __float_as_uint(rest) & 0xFFFF0000u;
            p[n][i] = __builtin_bit_cast(__bf16, (unsigned short)(u >> 16));
            rest -= __uint_as_float(u);
        }
        p[N - 1][i] = (__bf16)rest;
    }
}

constexpr int kRing = 3;  // tiles of 32 tokens that each wave has in LDS
constexpr int kLift = 66;  // probabilities are taken 2^kLift times as large to be weighed
constexpr float kLifted = 0x1p66f;
template <int D>
constexpr int kTileBytes = 32 * D + 2 * D;  // keys, values, key scales, value scales

// A lane's share of 32 tokens as they lie in memory
template <int D>
struct Tile {
    unsigned k[2][D / 32];  // keys: D / 4 channels of two tokens
    unsigned v[D / 16];     // values: eight tokens of D / 16 channels
    unsigned vs[D / 16];    // the scale bytes of those tokens, [token][group]
    unsigned look;          // one word of vs for every lane of 16: together all of them
    unsigned char ks[2];    // the scale bytes of the keys' group
};

// 16 columns, `cols` to a piece: the sum over the pieces, in all of them
template <int COLS>
__device__ __forceinline__ float fold(float x) {
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xF, 0xF, true));
    if constexpr (COLS == 4) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x124, 0xF, 0xF, true));
    return x;
}

// JOINT: a workgroup's four waves take the tiles of one row and head in turn and add up in LDS (short rows: one launch);
// otherwise every wave is a worker of its own.
// COLS < 16: no more queries than that, whose pieces (two of fp16, up to four of fp32) take the other columns, which a product
// computes anyway: one product instead of one for each piece, and the columns are added up, of the scores for each tile, of the
// output at the end.
template <int TYPE, int D, int NM, bool COUNT, bool JOINT, int COLS>
__global__ __launch_bounds__(256) void kv4_attend_kernel(AttendArgs a) {
    using T = typename Elem<TYPE>::T;
    constexpr int PIECES = COLS < 16 ? 16 / COLS : TYPE == AFTER_T_BF16 ? 1 : TYPE == AFTER_T_F16 ? 2 : 3;
    constexpr int NP = COLS < 16 ? 1 : PIECES;  // operands of a lane
    constexpr int G = D / 32, S = D / 32, KW = D / 32, VW = D / 16;  // groups, steps of a score, dwords of keys / values per lane
    constexpr int RING = kRing, BYTES = kTileBytes<D>, LOADS = D / 32 + 1;
    constexpr int STRIDE = JOINT ? 128 : 32;  // tokens from one tile of a wave to its next
    extern __shared__ __align__(16) char lds[];  // [4][RING][BYTES]; JOINT: then [4][16][D + 4] floats
    const after_kv4& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, kq = lane >> 4;
    const int col = l15 % COLS, piece_of = l15 / COLS;  // this lane's query of each 16, and which piece of it
    // the first row and head of this worker's share, and where in it the share begins
    const int worker = blockIdx.x * 4 + wave;
    int r, h, step = 0;
    long long left = 1;
    if constexpr (JOINT) {
        r = blockIdx.x / c.kv_heads;
        h = blockIdx.x % c.kv_heads;
    } else {
        long long all = 0;
        for (int i = lane; i < c.rows; i += 64) all += row_steps(c, i);
        all = wave_sum(all);
        const long long share = (all * c.kv_heads + a.workers - 1) / a.workers, at = share * worker;
        const long long mine = min(share, all * c.kv_heads - at);
        if (mine <= 0) return;
        left = (long long)__builtin_amdgcn_readfirstlane((int)(mine >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)mine);
        // (at < all * H, which the last row's sum reaches, unless another call changes the lengths meanwhile: that is the caller's
        // mistake, but here, in the join and in eviction every index stays in its range all the same, and every search ends)
        long long before = 0;
        int n = 0;
        r = -1;
        for (int r0 = 0; r0 < c.rows; r0 += 64) {
            const int own = r0 + lane < c.rows ? row_steps(c, r0 + lane) : 0;
            long long sum = own;
#pragma unroll
            for (int o = 1; o < 64; o *= 2) {
                const long long y = __shfl_up(sum, o);
                if (lane >= o) sum += y;
            }
            const unsigned long long past = __ballot((before + sum) * c.kv_heads > at);
            if (past) {
                const int first = __ffsll(past) - 1;
                r = r0 + first;
                n = __shfl(own, first);
                before += first ? __shfl(sum, first - 1) : 0;
                break;
            }
            before += __shfl(sum, 63);
        }
        if (r < 0) return;
        const long long in = at - before * c.kv_heads;
        h = (int)(in / n);
        step = (int)(in - (long long)h * n);
        // (the same in every lane: kept in scalar registers)
        r = __builtin_amdgcn_readfirstlane(r);
        h = __builtin_amdgcn_readfirstlane(h);
        step = __builtin_amdgcn_readfirstlane(step);
    }

    for (;;) {  // one piece of the share: slots of one row and head
    const int len = row_length(c, r), steps = (len + kStep - 1) / kStep, rh = r * c.kv_heads + h;
    const int n_steps = JOINT ? steps : (int)min(left, (long long)(steps - step));
    const int begin = step * kStep, end = min((step + n_steps) * kStep, len);
    const bool whole = n_steps == steps;

    bf16x8 qf[NM][S][NP];
    int vis[NM];
#pragma unroll
    for (int nm = 0; nm < NM; ++nm) {
        const int m = nm * 16 + col, t = m / a.group, g = m - t * a.group;
        const bool in = m < a.m_rows;
        vis[nm] = in ? max(len - a.tokens + t + 1, 0) : 0;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float y[8] = {};
            if (in) load_n<8, T>((const T*)a.q + r * a.qrs + t * a.qts + (long long)(h * a.group + g) * a.qhs + D / 4 * kq + 8 * s, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] *= a.q_sign;
            if constexpr (COLS < 16) {
                bf16x8 z[PIECES];
                query_pieces8<PIECES>(y, z);
                qf[nm][s][0] = z[0];
#pragma unroll
                for (int q = 1; q < PIECES; ++q)
                    if (piece_of == q) qf[nm][s][0] = z[q];
            } else
                query_pieces8<NP>(y, qf[nm][s]);
        }
    }
    const int all_see = len - a.tokens + 1;  // slots below this are seen by every query

    f32x4 o[NM][2 * G];
    float mx[NM], l[NM];
    float off[NM], times[NM], limit[NM];  // p = 2^(score times - off); the maximum moves beyond the limit
#pragma unroll
    for (int nm = 0; nm < NM; ++nm) {
        mx[nm] = limit[nm] = -INFINITY;
        l[nm] = 0.f;
        off[nm] = 0.f, times[nm] = a.scale2;
#pragma unroll
        for (int i = 0; i < 2 * G; ++i) o[nm][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    const size_t base = (size_t)rh * c.capacity;
    // 32 tokens at a time go from memory to this wave's own ring in LDS, without passing registers: two tiles are on their way
    // while one is computed (the memory's latency is longer than a tile's work), and no wave waits for another.
    const unsigned ring = (unsigned)(unsigned long)(__attribute__((address_space(3))) char*)lds + wave * (RING * BYTES);
    const unsigned char* sc_at = (lane < 8 * G ? c.key_scales : c.value_scales - 32 * G) + base * G + lane * 4;  // keys' scales, then the values'
    auto fetch = [&](int t0, int slot) {
        const unsigned to = ring + slot * BYTES;
        const unsigned long long k = reinterpret_cast<unsigned long long>(c.keys + (base + t0) * (D / 2));
        const unsigned long long v = reinterpret_cast<unsigned long long>(c.values + (base + t0) * (D / 2));
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            lds_dma16(to + i * 1024, lane * 16, k + i * 1024);
            lds_dma16(to + 16 * D + i * 1024, lane * 16, v + i * 1024);
        }
        if (lane < 16 * G)
            __builtin_amdgcn_global_load_lds((gbl_ptr_t)(sc_at + t0 * G), (lds_ptr_t)(__attribute__((address_space(3))) char*)(unsigned long)(to + 32 * D), 4, 0, 0);
    };
    int t0 = begin + (JOINT ? 32 * wave : 0);
#pragma unroll
    for (int i = 0; i < RING - 1; ++i)
        if (t0 + i * STRIDE < end) fetch(t0 + i * STRIDE, i);
    for (int slot = 0; t0 < end; t0 += STRIDE, slot = slot == RING - 1 ? 0 : slot + 1) {
        // (the slot that the tile before used is free once its values have been read)
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (t0 + (RING - 1) * STRIDE < end) {
            fetch(t0 + (RING - 1) * STRIDE, slot == 0 ? RING - 1 : slot - 1);
            wait_vmcnt_imm<(RING - 1) * LOADS>();
        } else if (RING == 3 && t0 + STRIDE < end)
            wait_vmcnt_imm<LOADS>();
        else
            wait_vmcnt_imm<0>();
        Tile<D> w;
        const char* at = lds + (wave * RING + slot) * BYTES;
        const int tok = 8 * (l15 >> 2) + (l15 & 3);  // tile rows (2 x 16): row m of half f is token 8 (m / 4) + 4 f + m % 4
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const unsigned* p = reinterpret_cast<const unsigned*>(at + (tok + 4 * f) * (D / 2) + kq * (D / 8));
#pragma unroll
            for (int i = 0; i < KW; ++i) w.k[f][i] = p[i];
            w.ks[f] = at[32 * D + (tok + 4 * f) * G + kq * G / 4];
        }
        {
            const unsigned* p = reinterpret_cast<const unsigned*>(at + 16 * D + kq * (4 * D) + l15 * (D / 4));
#pragma unroll
            for (int i = 0; i < VW; ++i) w.v[i] = p[i];
            const unsigned* ps = reinterpret_cast<const unsigned*>(at + 32 * D + 32 * G + kq * (8 * G));
#pragma unroll
            for (int i = 0; i < 2 * G; ++i) w.vs[i] = ps[i];
            w.look = ps[l15 % (2 * G)];
        }
        f32x4 sc[NM][2];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
#pragma unroll
            for (int nm = 0; nm < NM; ++nm) sc[nm][f] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const bf16x8 kf = widen8(w.k[f][s], byte_scale(w.ks[f]));
#pragma unroll
                for (int nm = 0; nm < NM; ++nm)
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p) sc[nm][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[nm][s][p], sc[nm][f], 0, 0, 0);
            }
        }
        if constexpr (COLS < 16) {
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[0][f][i] = fold<COLS>(sc[0][f][i]);
        }
        __builtin_amdgcn_sched_barrier(0);
        const bool masked = t0 + 32 > all_see;
        if (masked) {
#pragma unroll
            for (int nm = 0; nm < NM; ++nm)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (t0 + 8 * kq + j >= vis[nm]) sc[nm][j >> 2][j & 3] = -INFINITY;
        }
        float p[NM][8];
#pragma unroll
        for (int nm = 0; nm < NM; ++nm) {
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, sc[nm][j >> 2][j & 3]);
            if constexpr (COUNT) {
                const int m = nm * 16 + col;
                if (m < a.m_rows && piece_of == 0) {
                    float* to = a.scores + ((size_t)rh * a.m_rows + m) * c.capacity + t0 + 8 * kq;
                    *reinterpret_cast<f32x4*>(to) = sc[nm][0];
                    *reinterpret_cast<f32x4*>(to + 4) = sc[nm][1];
                }
            }
            // The maximum moves only when a score outgrows it by 2^2, so that most tiles need no exchange between lanes: a
            // probability of up to 4 is as exact.  Where it is beyond kFarTop, scores are brought down here in every tile: the usual
            // one has no branch for it.
            top *= a.scale2;
            if (__any(top > limit[nm])) {
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float now = fmaxf(mx[nm], top), f = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx[nm] - now);
                const float below = now == -INFINITY ? 0.f : now;
                const bool far = __any(fabsf(below) > kFarTop);
                mx[nm] = now;
                off[nm] = far ? 0.f : below, times[nm] = far ? 1.f : a.scale2, limit[nm] = far ? -INFINITY : now + 2.f;
                l[nm] *= f;
#pragma unroll
                for (int i = 0; i < 2 * G; ++i) o[nm][i] = o[nm][i] * f;
                if (far) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) sc[nm][j >> 2][j & 3] = scaled_below(sc[nm][j >> 2][j & 3], a.scale2, below);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[nm][j] = __builtin_amdgcn_exp2f(fmaf(sc[nm][j >> 2][j & 3], times[nm], -off[nm]));
                l[nm] += p[nm][j];
            }
        }
        // P times the scale of its token and group, as bf16 pieces.  The scale is a power of two: its exponent is added to the
        // probability's as an integer, two tokens at a time -- one v_perm_b32 for both bytes, one v_pk_mad_u16, and a maximum
        // with 0 for what falls below bf16's exponents (products below 2^-126 vanish): a third of the instructions of extracting
        // eight scales per group and multiplying.  With p taken 2^kLift times as large, a p of 0 stays below them under every
        // scale less than 2^65; larger ones are multiplied.  Pieces are cut off, not rounded, so that none is negative; a single
        // one is rounded.
        u16x2 bits[NM][NP][4];
#pragma unroll
        for (int nm = 0; nm < NM; ++nm)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x0 = p[nm][2 * i] * kLifted, x1 = p[nm][2 * i + 1] * kLifted;
#pragma unroll
                for (int q = 0; COLS < 16 && q < PIECES - 1; ++q) {  // what this lane's piece leaves to the ones before it
                    const unsigned taken = piece_of > q ? 0xFFFF0000u : 0u;
                    x0 -= __uint_as_float(__float_as_uint(x0) & taken);
                    x1 -= __uint_as_float(__float_as_uint(x1) & taken);
                }
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    unsigned u;
                    if constexpr (PIECES == 1)
                        u = __builtin_bit_cast(unsigned, bf16x2{(__bf16)x0, (__bf16)x1});
                    else
                        u = __builtin_amdgcn_perm(__float_as_uint(x1), __float_as_uint(x0), 0x07060302u);
                    x0 -= __uint_as_float(u << 16);
                    x1 -= __uint_as_float(u & 0xFFFF0000u);
                    bits[nm][q][i] = __builtin_bit_cast(u16x2, u) - (unsigned short)((127 + kLift) << 7);
                }
            }
        const bool special = masked || __any(w.look & w.look << 1 & 0x80808080u);  // (bytes from 192 on: the two highest bits)
#pragma unroll
        for (int g = 0; g < G; ++g) {
            u32x4 pf[NM][NP];
            if (special) {
                // (a slot that is not seen, a large scale, or a NaN group, whatever its codes: what a masked slot holds must not reach
                // the sum, 0 x NaN would; all ones or none by a shift, since the compiler branches around a choice)
#pragma unroll
                for (int nm = 0; nm < NM; ++nm) {
                    float y[8];
                    bf16x8 z[PIECES];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const unsigned b = w.vs[(j * G + g) >> 2] >> 8 * ((j * G + g) & 3) & 255u;
                        y[j] = __uint_as_float(__float_as_uint(p[nm][j] * scale_or_nan(b)) & (unsigned)(t0 + 8 * kq + j - vis[nm] >> 31));
                    }
                    pieces8<PIECES>(y, z);
#pragma unroll
                    for (int q = 0; q < PIECES; ++q)
                        if (NP > 1 || piece_of == q) pf[nm][NP > 1 ? q : 0] = __builtin_bit_cast(u32x4, z[q]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned b = G == 4 ? __builtin_amdgcn_perm(w.vs[2 * i + 1], w.vs[2 * i], 0x0C040C00u + 0x00010001u * g)
                                              : __builtin_amdgcn_perm(0u, w.vs[i], 0x0C020C00u + 0x00010001u * g);
#pragma unroll
                    for (int nm = 0; nm < NM; ++nm)
#pragma unroll
                        for (int q = 0; q < NP; ++q) {
                            s16x2 x;  // (the compiler takes a product by 128 apart into a shift and a sum)
                            asm("v_pk_mad_u16 %0, %1, %2, %3" : "=v"(x) : "v"(b), "s"(0x00800080u), "v"(bits[nm][q][i]));
                            pf[nm][q][i] = __builtin_bit_cast(unsigned, __builtin_elementwise_max(x, s16x2{0, 0}));
                        }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bf16x8 vf = widen8(w.v[2 * g + i], 1.f);
#pragma unroll
                for (int nm = 0; nm < NM; ++nm)
#pragma unroll
                    for (int q = NP - 1; q >= 0; --q)
                        o[nm][2 * g + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, __builtin_bit_cast(bf16x8, pf[nm][q]), o[nm][2 * g + i], 0, 0, 0);
            }
        }
    }

#pragma unroll
    for (int nm = 0; nm < NM; ++nm) {
        l[nm] += __shfl_xor(l[nm], 16);
        l[nm] += __shfl_xor(l[nm], 32);
        if constexpr (COLS < 16) {
#pragma unroll
            for (int i = 0; i < 2 * G; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nm][i][e] = fold<COLS>(o[nm][i][e]);
        }
    }
    if constexpr (JOINT) {  // the four waves' shares -> one
        __shared__ float sm[4][NM * 16], sl[4][NM * 16];
        float(*so)[16][D + 4] = reinterpret_cast<float(*)[16][D + 4]>(lds);
#pragma unroll
        for (int nm = 0; nm < NM; ++nm)
            if (kq == 0) {
                sm[wave][nm * 16 + l15] = mx[nm];
                sl[wave][nm * 16 + l15] = l[nm];
            }
#pragma unroll
        for (int nm = 0; nm < NM; ++nm) {
            __syncthreads();
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int e = 0; e < 8; ++e) so[wave][l15][32 * g + 8 * kq + e] = o[nm][2 * g + (e & 1)][e >> 1];
            __syncthreads();
            constexpr int W = D / 16;
            const int row = threadIdx.x >> 4, d = (threadIdx.x & 15) * W, m = nm * 16 + row;
            if (m < a.m_rows) {
                float top = -INFINITY, sum = 0.f, acc[W] = {};
                for (int w = 0; w < 4; ++w) top = fmaxf(top, sm[w][nm * 16 + row]);
                for (int w = 0; w < 4; ++w) {
                    const float mw = sm[w][nm * 16 + row];
                    const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - top);
                    // (a wave without a visible slot has sum 0; one whose scores were all NaN keeps its NaN: NaN x 0)
                    sum += sl[w][nm * 16 + row] * f;
#pragma unroll
                    for (int i = 0; i < W; ++i) acc[i] += so[w][row][d + i] * f;
                }
                const int t = m / a.group, g = m - t * a.group;
                const float inv = inverse_sum(sum, len - a.tokens + t + 1 > 0);
#pragma unroll
                for (int i = 0; i < W; ++i) acc[i] *= inv;
                store_n<W, T>((T*)a.out + (((size_t)r * a.tokens + t) * a.heads + h * a.group + g) * D + d, acc);
                if (COUNT && (threadIdx.x & 15) == 0) a.final_ml[(size_t)rh * a.m_rows + m] = f32x2{top, sum};
            }
        }
        return;
    } else {
        const size_t piece = (size_t)worker + rh;
        if (lane == 0) {
            if (step == 0) a.ends[rh].x = (int)piece;
            if (step + n_steps == steps) a.ends[rh].y = (int)piece;
        }
#pragma unroll
        for (int nm = 0; nm < NM; ++nm) {
            const int m = nm * 16 + col;
            if (m < a.m_rows && piece_of == 0) {
                if ((!whole || COUNT) && kq == 0) a.part_ml[piece * a.m_rows + m] = f32x2{mx[nm], l[nm]};
                const float inv = inverse_sum(l[nm], vis[nm] > 0);
                const int t = m / a.group, g0 = m - t * a.group;
                T* out = (T*)a.out + (((size_t)r * a.tokens + t) * a.heads + h * a.group + g0) * D + 8 * kq;
                float* part = a.part_o + (piece * a.m_rows + m) * D + 8 * kq;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = o[nm][2 * g + (e & 1)][e >> 1] * (whole ? inv : 1.f);
                    if (whole)
                        store_n<8, T>(out + 32 * g, y);
                    else
                        store_n<8, float>(part + 32 * g, y);
                }
            }
        }
        left -= n_steps;
        if (left <= 0) return;
        step = 0;
        if (++h == c.kv_heads) {
            h = 0;
            do {
                if (++r == c.rows) return;  // (work is left, so a later row holds it: as above)
            } while (row_length(c, r) == 0);
        }
    }
    }
}

// ---------------------------------------------------------------------------------------------------------------- many queries
// More than 32 queries of a row that share a head (a chunk of a prompt, the last tokens that say what is worth keeping): 128 of
// them per workgroup, 32 to a wave, over the same tiles of 64 tokens.  The tiles are widened to bf16 once for the four waves and
// kept in LDS in the order in which the matrix instructions take them (a lane's operand is 16 bytes at its own number: no
// conflicts); while one tile is multiplied the next one's codes are on their way in registers.
// What bounds it: waits between phases that depend on each other (one barrier a tile, codes asked for one tile ahead, scores, softmax
// and product one behind the other inside a wave): the matrix pipes are busy a quarter of the time, the vector unit less than half,
// and a wave waits 0.4 of its own.  32 tokens of 4 rows of 9001 .. 16384, bf16, 32 / 8 heads of 128: 52 us, 0.5 PFLOP/s, the join 10
// (64 KB of sums a piece), the weights, for which the scores are formed again, 38.5; 64 tokens of 64 / 8 heads over the same rows
// 207 and 23, 512 tokens 1163 and 60; 8 rows of 1 .. 16384: 151 us in all, 177 with equal splits of each row.
constexpr int kWideRows = 128, kWideTile = 64;

template <int D>
struct Raw {  // a thread's share of a tile as it lies in memory
    u32x4 k, v;
    unsigned vs[D / 16];
    unsigned char ks;
};

template <int D>
struct Widen {
    static constexpr int G = D / 32, USED = 2 * D;  // threads that hold a piece: 16 bytes of keys and 16 of values each
    static constexpr int KEYS = kWideTile * D * 2;  // bytes of a widened tile's keys; as many of its values
    const after_kv4& c;
    size_t base;
    int token, group;   // keys: one token's group of 32 channels
    int block, quad;    // values: four channels of eight tokens
    unsigned k_to, v_to;
    __device__ __forceinline__ Widen(const after_kv4& cache, int rh) : c(cache), base((size_t)rh * cache.capacity) {
        const int t = threadIdx.x % USED;
        token = t / G;
        group = t % G;
        // operand of half f of the 32 tokens: row m is token 8 (m / 4) + 4 f + m % 4; lane 16 kq + m holds channels 32 s + 8 kq ..
        k_to = ((((token >> 5) * 2 + (token >> 2 & 1)) * G + group) * 64 + ((token & 31) >> 3) * 4 + (token & 3)) * 16;
        block = t / (D / 4);
        quad = t % (D / 4);
        const int l15 = D == 128 ? quad >> 1 : quad, g0 = D == 128 ? 2 * (quad & 1) : 0;
        // operand (g, i): row l15 is channel 32 g + 2 l15 + i; lane 16 kq + l15 holds tokens 8 kq ..
        v_to = KEYS + (((block >> 2) * 2 * G + 2 * g0) * 64 + (block & 3) * 16 + l15) * 16;
    }
    __device__ __forceinline__ bool mine() const { return USED == 256 || threadIdx.x < USED; }
    // (a tile may reach past the last 32 slots that are in use: capacity is a multiple of 32)
    __device__ __forceinline__ void load_keys(Raw<D>& w, int t0) const {
        const size_t at = base + min(t0 + token, c.capacity - 1);
        w.k = *reinterpret_cast<const u32x4*>(c.keys + at * (D / 2) + 16 * group);
        w.ks = c.key_scales[at * G + group];
    }
    __device__ __forceinline__ void load_values(Raw<D>& w, int t0) const {
        const size_t at = base + min(t0 + 8 * block, c.capacity - 8);
        w.v = *reinterpret_cast<const u32x4*>(c.values + at / 8 * (4 * D) + 16 * quad);
        const unsigned* ps = reinterpret_cast<const unsigned*>(c.value_scales + at * G);
#pragma unroll
        for (int i = 0; i < 2 * G; ++i) w.vs[i] = ps[i];
    }
    __device__ __forceinline__ void store_keys(const Raw<D>& w, char* lds) const {
        const float sc = byte_scale(w.ks);
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<bf16x8*>(lds + k_to + i * 256) = widen8(w.k[i], sc);
    }
    // A NaN group is left out, its token marked in bad[g]: the queries that see it get their NaN apart from the product, in which
    // it would reach all of them.  So is any scale beyond the format's, which slots behind the row's length may hold: nobody sees
    // them, but their codes times 2^126 would be infinities.
    __device__ __forceinline__ void store_values(const Raw<D>& w, char* lds, unsigned long long* bad) const {
        const int g0 = D == 128 ? 2 * (quad & 1) : 0;
#pragma unroll
        for (int gg = 0; gg < 2; ++gg) {
            float sc[8];
            bool any = false;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int byte = j * G + g0 + gg;
                const unsigned b = w.vs[G == 4 ? j : j >> 1] >> 8 * (byte & 3) & 255u;
                any |= b > kMaxByte;
                sc[j] = byte_scale(b);
            }
            if (any) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (sc[j] > byte_scale(kMaxByte)) {
                        atomicOr(&bad[g0 + gg], 1ull << (8 * block + j));
                        sc[j] = 1.f;  // (any that keeps its codes finite)
                    }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const unsigned x = w.v[2 * gg + i];
                auto pair = [&](bf16x2 lo, bf16x2 hi) { return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, hi), __builtin_bit_cast(unsigned, lo), 0x07060100u); };
                u32x4 y;
                y[0] = pair(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, sc[0], 0), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, sc[1], 0));
                y[1] = pair(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, sc[2], 1), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, sc[3], 1));
                y[2] = pair(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, sc[4], 2), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, sc[5], 2));
                y[3] = pair(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, sc[6], 3), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, sc[7], 3));
                *reinterpret_cast<u32x4*>(lds + v_to + (2 * gg + i) * 1024) = y;
            }
        }
    }
};

// the wave's 32 queries as operands: qf[nm][s][piece], channels 32 s + 8 kq ..; vis: the slots that each sees
template <int TYPE, int D, int NP>
__device__ __forceinline__ void load_queries(const AttendArgs& a, int r, int h, int m0, int len, bf16x8 (&qf)[2][D / 32][NP], int (&vis)[2]) {
    using T = typename Elem<TYPE>::T;
    const int lane = threadIdx.x & 63, l15 = lane & 15, kq = lane >> 4;
#pragma unroll
    for (int nm = 0; nm < 2; ++nm) {
        const int m = m0 + nm * 16 + l15, t = m / a.group, g = m - t * a.group;
        const bool in = m < a.m_rows;
        vis[nm] = in ? max(len - a.tokens + t + 1, 0) : 0;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            float y[8] = {};
            if (in) load_n<8, T>((const T*)a.q + r * a.qrs + t * a.qts + (long long)(h * a.group + g) * a.qhs + 32 * s + 8 * kq, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] *= a.q_sign;
            query_pieces8<NP>(y, qf[nm][s]);
        }
    }
}

// scores of 32 tokens.  BY_TOKEN: sc[nm][f][i] is query l15 (a column), token 8 kq + 4 f + i; otherwise query 4 kq + i, token
// 8 (l15 / 4) + 4 f + l15 % 4 (a column): the operands are alike, only their order differs.
template <int D, int NP, bool BY_TOKEN>
__device__ __forceinline__ void scores32(const char* keys, const bf16x8 (&qf)[2][D / 32][NP], f32x4 (&sc)[2][2]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int f = 0; f < 2; ++f) {
        sc[0][f] = sc[1][f] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            const bf16x8 kf = *reinterpret_cast<const bf16x8*>(keys + ((f * (D / 32) + s) * 64 + lane) * 16);
#pragma unroll
            for (int nm = 0; nm < 2; ++nm)
#pragma unroll
                for (int p = NP - 1; p >= 0; --p)
                    sc[nm][f] = BY_TOKEN ? __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[nm][s][p], sc[nm][f], 0, 0, 0)
                                         : __builtin_amdgcn_mfma_f32_16x16x32_bf16(qf[nm][s][p], kf, sc[nm][f], 0, 0, 0);
        }
    }
}

// The tiles of all rows are shared out over the workgroups of a head in pieces of one length, the least with which rows x splits
// workgroups do (each row's last piece may be shorter): with rows of different lengths all end at about the same time.
struct WidePiece {
    int row, at, of;  // the at-th of the row's `of` pieces
    int first;        // its number among the head's
    int slots;        // of a piece
};
__device__ __forceinline__ int wide_tiles(const after_kv4& c, int r) { return (row_length(c, r) + kWideTile - 1) / kWideTile; }
__device__ __forceinline__ bool find_piece(const after_kv4& c, int splits, int unit, WidePiece& p) {
    const int lane = threadIdx.x & 63, units = c.rows * splits;
    int share = 1 << 24;  // (one piece to a row)
    if (splits > 1) {
        long long all = 0;
        for (int i = lane; i < c.rows; i += 64) all += wide_tiles(c, i);
        // (a row's last piece: at most one more for each)
        share = (int)max(1ll, (wave_sum(all) + units - c.rows - 1) / (units - c.rows));
    }
    int before = 0;
    for (int r0 = 0; r0 < c.rows; r0 += 64) {
        const int n = r0 + lane < c.rows ? (wide_tiles(c, r0 + lane) + share - 1) / share : 0, sum = lane_sums(n);
        const unsigned long long past = __ballot(before + sum > unit);
        if (past) {
            const int j = __ffsll(past) - 1;
            p.row = __builtin_amdgcn_readfirstlane(r0 + j);
            p.of = __builtin_amdgcn_readlane(n, j);
            p.first = __builtin_amdgcn_readfirstlane(before) + __builtin_amdgcn_readlane(sum, j) - p.of;
            p.at = unit - p.first;
            p.slots = __builtin_amdgcn_readfirstlane(share) * kWideTile;
            return true;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

template <int TYPE, int D>
__global__ __launch_bounds__(256, TYPE == AFTER_T_F32 ? 1 : 2) void kv4_wide_kernel(AttendArgs a, int splits, int mgroups) {
    using T = typename Elem<TYPE>::T;
    constexpr int NP = TYPE == AFTER_T_BF16 ? 1 : TYPE == AFTER_T_F16 ? 2 : 3;
    constexpr int G = D / 32, STAGE = 2 * Widen<D>::KEYS;
    extern __shared__ __align__(16) char lds[];
    __shared__ unsigned long long bad[3][G];
    const after_kv4& c = a.c;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, kq = lane >> 4;
    // (neighbours are dispatched to different XCDs: the workgroups that read one piece of the cache stand eight apart, on one L2)
    const int x = blockIdx.x, mg = (x >> 3) % mgroups, unit = (x >> 3) / mgroups * 8 + (x & 7), n_rh = c.rows * c.kv_heads;
    if (unit >= n_rh * splits) return;
    const int h = unit % c.kv_heads, units = c.rows * splits;
    WidePiece w;
    if (!find_piece(c, splits, unit / c.kv_heads, w)) return;
    const int r = w.row, rh = r * c.kv_heads + h, len = row_length(c, r), used = w.of, first = h * units + w.first;
    if (mg == 0 && w.at == 0 && threadIdx.x == 0) a.ends[rh] = int2{first, first + used - 1};
    const int m0 = mg * kWideRows + wave * 32;
    const int begin = w.at * w.slots, last_m = min((mg + 1) * kWideRows, a.m_rows) - 1;
    const int end = min(min(begin + w.slots, len), len - a.tokens + last_m / a.group + 1);  // (what the last query here sees)
    const int all_see = len - a.tokens + m0 / a.group + 1;                      // every query of the wave sees the slots below

    bf16x8 qf[2][G][NP];
    int vis[2];
    load_queries<TYPE, D, NP>(a, r, h, m0, len, qf, vis);
    f32x4 o[2][2 * G];
    float mx[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float off[2] = {0.f, 0.f}, times[2] = {a.scale2, a.scale2}, limit[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nm = 0; nm < 2; ++nm)
#pragma unroll
        for (int i = 0; i < 2 * G; ++i) o[nm][i] = f32x4{0.f, 0.f, 0.f, 0.f};

    const Widen<D> widen(c, rh);
    Raw<D> raw;
    if (threadIdx.x < 3 * G) bad[threadIdx.x / G][threadIdx.x % G] = 0;
    if (begin < end && widen.mine()) {
        widen.load_keys(raw, begin);
        widen.load_values(raw, begin);
    }
    __syncthreads();
    int n = 0;
    for (int t0 = begin; t0 < end; t0 += kWideTile, ++n) {
        char* stage = lds + (n & 1) * STAGE;
        if (widen.mine()) {
            widen.store_keys(raw, stage);
            widen.store_values(raw, stage, bad[n % 3]);
        }
        __syncthreads();  // (one for each tile: the other stage was read before the last one)
        if (threadIdx.x < G) bad[(n + 2) % 3][threadIdx.x] = 0;  // (read before this barrier, written again after the next)
        if (t0 + kWideTile < end && widen.mine()) {
            widen.load_keys(raw, t0 + kWideTile);
            widen.load_values(raw, t0 + kWideTile);
        }
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            const char* keys = stage + part * (Widen<D>::KEYS / 2);
            const char* values = stage + Widen<D>::KEYS + part * (Widen<D>::KEYS / 2);
            const int s0 = t0 + 32 * part;
            f32x4 sc[2][2];
            scores32<D, NP, true>(keys, qf, sc);
            if (s0 + 32 > all_see) {
#pragma unroll
                for (int nm = 0; nm < 2; ++nm)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (s0 + 8 * kq + j >= vis[nm]) sc[nm][j >> 2][j & 3] = -INFINITY;
            }
            bf16x8 pf[2][NP];
#pragma unroll
            for (int nm = 0; nm < 2; ++nm) {
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, sc[nm][j >> 2][j & 3]);
                top *= a.scale2;
                if (__any(top > limit[nm])) {  // (as in attend_packed: the maximum moves when scores outgrow it by 2^8)
                    top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const float now = fmaxf(mx[nm], top), f = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx[nm] - now);
                    const float below = now == -INFINITY ? 0.f : now;
                    const bool far = __any(fabsf(below) > kFarTop);
                    mx[nm] = now;
                    off[nm] = far ? 0.f : below, times[nm] = far ? 1.f : a.scale2, limit[nm] = far ? -INFINITY : now + 8.f;
                    l[nm] *= f;
#pragma unroll
                    for (int i = 0; i < 2 * G; ++i) o[nm][i] = o[nm][i] * f;
                    if (far) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) sc[nm][j >> 2][j & 3] = scaled_below(sc[nm][j >> 2][j & 3], a.scale2, below);
                    }
                }
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p[j] = __builtin_amdgcn_exp2f(fmaf(sc[nm][j >> 2][j & 3], times[nm], -off[nm]));
                    l[nm] += p[j];
                }
                pieces8<NP>(p, pf[nm]);
            }
#pragma unroll
            for (int i = 0; i < 2 * G; ++i) {
                const bf16x8 vf = *reinterpret_cast<const bf16x8*>(values + (i * 64 + lane) * 16);
#pragma unroll
                for (int nm = 0; nm < 2; ++nm)
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p) o[nm][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[nm][p], o[nm][i], 0, 0, 0);
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const unsigned long long marked = bad[n % 3][g];
            if (marked) {
#pragma unroll
                for (int nm = 0; nm < 2; ++nm) {
                    const int sees = vis[nm] - t0;
                    if (sees > 0 && (marked & (sees >= 64 ? ~0ull : (1ull << sees) - 1))) o[nm][2 * g] = o[nm][2 * g + 1] = f32x4{NAN, NAN, NAN, NAN};
                }
            }
        }
    }

    const size_t piece = (size_t)first + w.at;
#pragma unroll
    for (int nm = 0; nm < 2; ++nm) {
        l[nm] += __shfl_xor(l[nm], 16);
        l[nm] += __shfl_xor(l[nm], 32);
        const int m = m0 + nm * 16 + l15;
        if (m >= a.m_rows) continue;
        if (kq == 0) a.part_ml[piece * a.m_rows + m] = f32x2{mx[nm], l[nm]};
        const bool whole = used == 1;
        const float inv = whole ? inverse_sum(l[nm], vis[nm] > 0) : 1.f;
        const int t = m / a.group, g0 = m - t * a.group;
        T* out = (T*)a.out + (((size_t)r * a.tokens + t) * a.heads + h * a.group + g0) * D + 8 * kq;
        float* part = a.part_o + (piece * a.m_rows + m) * D + 8 * kq;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = o[nm][2 * g + (e & 1)][e >> 1] * inv;
            if (whole)
                store_n<8, T>(out + 32 * g, y);
            else
                store_n<8, float>(part + 32 * g, y);
        }
    }
}

// (largest score, sum of exponentials to it) of query m over the pieces of a row and head, in every lane of the wave
__device__ __forceinline__ f32x2 join_ml(const AttendArgs& a, int2 p, int m) {
    const f32x2* ml = a.part_ml + m;
    float top = -INFINITY, sum = 0.f;
    for (int s = p.x + (int)(threadIdx.x & 63); s <= p.y; s += 64) {
        const f32x2 x = ml[(size_t)s * a.m_rows];
        const float now = fmaxf(top, x[0]);
        sum = (now == top ? sum : sum * __builtin_amdgcn_exp2f(top - now)) + x[1] * (x[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x[0] - now));
        top = now;
    }
    float all = top;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) all = fmaxf(all, __shfl_xor(all, o));
    sum *= top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top - all);  // (a sum without a maximum is 0 or NaN)
#pragma unroll
    for (int o = 1; o < 64; o *= 2) sum += __shfl_xor(sum, o);
    return f32x2{all, sum};
}

// The rows and heads that were cut into pieces -> the output, and zeros for empty rows.  One workgroup per row, head and query: a
// long row is cut into up to all workers, so 16 groups of 16 lanes share its pieces.
template <int TYPE, int D>
__global__ __launch_bounds__(256) void kv4_join_kernel(AttendArgs a) {
    using T = typename Elem<TYPE>::T;
    constexpr int W = D / 16;
    __shared__ float part[16][D];
    const after_kv4& c = a.c;
    const int rh = blockIdx.x / a.m_rows, m = blockIdx.x % a.m_rows, r = rh / c.kv_heads, h = rh % c.kv_heads;
    const int group = threadIdx.x >> 4, d = (threadIdx.x & 15) * W;
    const int2 ends = a.ends[rh], p = {max(ends.x, 0), min(ends.y, a.pieces - 1)};  // (an empty row has none: not looked at)
    float acc[W] = {};
    if (row_length(c, r) > 0) {
        if (p.x == p.y && !a.final_ml) return;  // (whole: written already)
        const f32x2 all = join_ml(a, p, m);
        if (a.final_ml && threadIdx.x == 0) a.final_ml[blockIdx.x] = all;
        if (p.x == p.y) return;
        const float inv = inverse_sum(all[1], row_length(c, r) - a.tokens + m / a.group + 1 > 0);
#pragma unroll 4
        for (int s = p.x + group; s <= p.y; s += 16) {
            const size_t at = (size_t)s * a.m_rows + m;
            const float ms = a.part_ml[at][0], f = (ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - all[0])) * inv;
            float x[W];
            load_n<W, float>(a.part_o + at * D + d, x);
#pragma unroll
            for (int i = 0; i < W; ++i) acc[i] += x[i] * f;
        }
    }
    store_n<W, float>(&part[group][d], acc);
    __syncthreads();
    if (threadIdx.x < D) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += part[i][threadIdx.x];
        const int t = m / a.group, g = m - t * a.group;
        ((T*)a.out)[(((size_t)r * a.tokens + t) * a.heads + h * a.group + g) * D + threadIdx.x] = (T)sum;
    }
}

// The probabilities that each slot received, from the stored scores: 1024 slots of one row and head, up to 32 queries.
__global__ __launch_bounds__(256) void kv4_weights_kernel(AttendArgs a, int slot_blocks, float decay) {
    const after_kv4& c = a.c;
    const int rh = blockIdx.x / slot_blocks, r = rh / c.kv_heads;
    const int len = row_length(c, r), s = (blockIdx.x % slot_blocks) * 1024 + 4 * threadIdx.x;
    if (s >= len) return;
    const f32x2* ml = a.final_ml + (size_t)rh * a.m_rows;
    const float* scores = a.scores + (size_t)rh * a.m_rows * c.capacity + s;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    int sees = len - a.tokens + 1, g = 0;  // slots that query m sees
#pragma unroll 8
    for (int m = 0; m < a.m_rows; ++m) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(scores + (size_t)m * c.capacity);
        const float top = ml[m][0], off = top == -INFINITY ? 0.f : top, inv = inverse_sum(ml[m][1], sees > 0);
        const bool far = fabsf(off) > kFarTop;
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // (rounded as where they were summed up: the probabilities add up to 1)
            const float y = far ? scaled_below(x[i], a.scale2, off) : fmaf(x[i], a.scale2, -off);
            sum[i] += s + i < sees ? __builtin_amdgcn_exp2f(y) * inv : 0.f;
        }
        if (++g == a.group) {
            g = 0;
            ++sees;
        }
    }
    float* w = c.weights + (size_t)rh * c.capacity + s;
    // (the four slots are inside the capacity; those past the length keep what they hold)
    if (s + 3 < len) {
        f32x4 old = {0.f, 0.f, 0.f, 0.f};
        if (decay != 0.f) old = *reinterpret_cast<const f32x4*>(w);
#pragma unroll
        for (int i = 0; i < 4; ++i) old[i] = decay == 0.f ? sum[i] : fmaf(decay, old[i], sum[i]);
        *reinterpret_cast<f32x4*>(w) = old;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (s + i < len) w[i] = decay == 0.f ? sum[i] : fmaf(decay, w[i], sum[i]);
    }
}

// ... for more than 32 queries: the scores are formed again (68 bytes of keys per slot, where storing and reading 33 scores is
// 264), up to 1024 slots of one row and head to a workgroup (its beginning costs as much as some 300), 32 queries to a wave.
constexpr int kWideSlots = 1024;  // at most
template <int TYPE, int D>
__global__ __launch_bounds__(256, TYPE == AFTER_T_F32 ? 1 : 2) void kv4_wide_weights_kernel(AttendArgs a, int slot_blocks, int slots, float decay) {
    constexpr int NP = TYPE == AFTER_T_BF16 ? 1 : TYPE == AFTER_T_F16 ? 2 : 3;
    constexpr int G = D / 32;
    extern __shared__ __align__(16) char lds[];  // two stages of keys
    __shared__ float sums[4][kWideSlots];
    const after_kv4& c = a.c;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, kq = lane >> 4;
    const int rh = blockIdx.x / slot_blocks, r = rh / c.kv_heads, h = rh % c.kv_heads;
    const int len = row_length(c, r), begin = (blockIdx.x % slot_blocks) * slots, end = min(begin + slots, len);
    if (begin >= end) return;
    const Widen<D> widen(c, rh);
    Raw<D> raw;
    for (int i = threadIdx.x; i < 4 * kWideSlots; i += 256) sums[i / kWideSlots][i % kWideSlots] = 0.f;
    int n = 0;
    for (int mg = 0; mg * kWideRows < a.m_rows; ++mg) {
        const int m0 = mg * kWideRows + wave * 32;
        bf16x8 qf[2][G][NP];
        int vis[2];
        load_queries<TYPE, D, NP>(a, r, h, m0, len, qf, vis);
        f32x2 ml = {0.f, 0.f};
        if (m0 + (lane & 31) < a.m_rows) ml = a.final_ml[(size_t)rh * a.m_rows + m0 + (lane & 31)];
        float off[2][4], inv[2][4];  // of query 16 nm + 4 kq + i
        int sees[2][4];
        bool far = false;
#pragma unroll
        for (int nm = 0; nm < 2; ++nm)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int m = nm * 16 + 4 * kq + i;
                const float top = __shfl(ml[0], m), sum = __shfl(ml[1], m);
                off[nm][i] = top == -INFINITY ? 0.f : top;
                far |= fabsf(off[nm][i]) > kFarTop;
                sees[nm][i] = __shfl(vis[nm], 4 * kq + i);
                inv[nm][i] = inverse_sum(sum, sees[nm][i] > 0);
            }
        far = __any(far);
        const int all_see = m0 + 32 <= a.m_rows ? len - a.tokens + m0 / a.group + 1 : 0;
        if (widen.mine()) widen.load_keys(raw, begin);
        for (int t0 = begin; t0 < end; t0 += kWideTile, ++n) {
            char* stage = lds + (n & 1) * Widen<D>::KEYS;
            if (widen.mine()) widen.store_keys(raw, stage);
            __syncthreads();
            if (t0 + kWideTile < end && widen.mine()) widen.load_keys(raw, t0 + kWideTile);
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                f32x4 sc[2][2];
                scores32<D, NP, false>(stage + part * (Widen<D>::KEYS / 2), qf, sc);
                if (far) {  // (as where they were summed up)
#pragma unroll
                    for (int nm = 0; nm < 2; ++nm)
#pragma unroll
                        for (int j = 0; j < 8; ++j) sc[nm][j >> 2][j & 3] = scaled_below(sc[nm][j >> 2][j & 3], a.scale2, off[nm][j & 3]);
                }
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                    const int tok = 32 * part + 8 * (l15 >> 2) + 4 * f + (l15 & 3), s = t0 + tok;
                    float w = 0.f;
#pragma unroll
                    for (int nm = 0; nm < 2; ++nm)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float x = __builtin_amdgcn_exp2f(far ? sc[nm][f][i] : fmaf(sc[nm][f][i], a.scale2, -off[nm][i]));
                            w = t0 + kWideTile <= all_see || s < sees[nm][i] ? fmaf(x, inv[nm][i], w) : w;
                        }
                    w += __shfl_xor(w, 16);
                    w += __shfl_xor(w, 32);
                    if (kq == f) sums[wave][t0 - begin + tok] += w;
                }
            }
        }
        __syncthreads();  // (the next group's first stage may be the one that is still read)
    }
    for (int s = begin + threadIdx.x; s < end; s += 256) {
        const int i = s - begin;
        const float sum = (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
        float* w = c.weights + (size_t)rh * c.capacity + s;
        *w = decay == 0.f ? sum : fmaf(decay, *w, sum);
    }
}

// ---------------------------------------------------------------------------------------------------------------- evict
// A key that orders floats as unsigned numbers, NaN below everything
__device__ __forceinline__ unsigned order_key(float x) {
    const unsigned u = __float_as_uint(x);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0u;
    return u == 0x80000000u ? 0x80000000u : (u >> 31) ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64, kSelLoads = 8, kSelSpan = 4 * kSelLoads * kSelThreads;

// One workgroup per (row, head): which slots stay, in order.  The `recent` newest stay; of the others the `want` with the
// largest weights.  The value of the smallest of those is found eleven bits at a time: a histogram of the next digit of the
// candidates (in four copies: a few digits hold most of the weights, and the same address twice in an instruction costs twice),
// and where from the top its sums pass `want`.  Then every thread counts what stays of its slots, the counts are summed up over
// lanes, waves and loads, and the slots are written: those above the value, and the first `want` equal to it.  A row of up to
// 32768 weights is read once and stays in registers.  64 rows of 20001 .. 32768: 25.1 us,
// 24 of 400 .. 1000: 7.2.
__global__ __launch_bounds__(kSelThreads) void kv4_select_kernel(after_kv4 c, int keep, int recent, int* slots) {
    __shared__ int4 hist[2048];
    __shared__ int tmp[kSelWaves];
    __shared__ int found[3];
    __shared__ int2 counts[kSelLoads * kSelWaves];
    const int rh = blockIdx.x, r = rh / c.kv_heads, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int len = row_length(c, r);
    int* out = slots + (size_t)rh * keep;
    const float* w = c.weights + (size_t)rh * c.capacity;
    for (int i = min(len, keep) + tid; i < keep; i += kSelThreads) out[i] = -1;
    if (len <= keep) {
        for (int i = tid; i < len; i += kSelThreads) out[i] = i;
        return;
    }
    const int old = len - recent;  // (recent <= keep < len)
    int want = keep - recent;      // (< old)
    for (int i = tid; i < recent; i += kSelThreads) out[want + i] = old + i;
    if (want == 0) return;

    u32x4 k[kSelLoads];
    auto load = [&](int i0) {
#pragma unroll
        for (int u = 0; u < kSelLoads; ++u) {
            const int i = i0 + 4 * tid + u * 4 * kSelThreads;  // (rows of weights begin and end at multiples of 128 bytes)
            if (i < old) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(w + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) k[u][j] = order_key(x[j]);
            }
        }
    };
    unsigned prefix = 0;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11, bins = 1 << bits;
        for (int i = tid; i < bins; i += kSelThreads) hist[i] = int4{0, 0, 0, 0};
        if (pass == 0) load(0);
        __syncthreads();
        for (int i0 = 0; i0 < old; i0 += kSelSpan) {
            if (old > kSelSpan && (pass > 0 || i0 > 0)) load(i0);
#pragma unroll
            for (int u = 0; u < kSelLoads; ++u) {
                if (i0 + u * 4 * kSelThreads >= old) break;  // (uniform)
                bool in[4];
                bool any = false;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    in[j] = i0 + 4 * tid + u * 4 * kSelThreads + j < old && (pass == 0 || (k[u][j] ^ prefix) >> shift < (unsigned)bins);
                    any |= in[j];
                }
                if (pass == 0 || __any(any)) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (in[j]) atomicAdd(reinterpret_cast<int*>(hist) + (k[u][j] >> shift & (bins - 1)) * 4 + (lane & 3), 1);
                }
            }
        }
        __syncthreads();
        // thread t looks at two bins (one, in the last pass), from the top
        const int per = bins / kSelThreads;
        int mine = 0, bin_sum[2] = {0, 0};
        for (int j = 0; j < per; ++j) {
            const int4 n = hist[bins - 1 - (tid * per + j)];
            bin_sum[j] = (n.x + n.y) + (n.z + n.w);
            mine += bin_sum[j];
        }
        int upto = lane_sums(mine);
        if (lane == 63) tmp[wave] = upto;
        __syncthreads();
        for (int v = 0; v < wave; ++v) upto += tmp[v];
        if (upto >= want && upto - mine < want) {
            const int above = upto - mine, second = above + bin_sum[0] < want;
            found[0] = bins - 1 - (tid * per + second);
            found[1] = want - above - (second ? bin_sum[0] : 0);
            found[2] = second ? bin_sum[1] : bin_sum[0];
        }
        __syncthreads();
        prefix |= (unsigned)found[0] << shift;
        want = found[1];  // of those equal to the prefix so far (the next write of `found` is three barriers on)
        if (want == found[2]) {  // all of them, as a rule the only one: what is not below them stays (never all: want < old)
            prefix -= 1;
            want = 0;
            break;
        }
    }

    int above = 0, equal = 0;  // before this span
    for (int i0 = 0; i0 < old; i0 += kSelSpan) {
        if (old > kSelSpan) load(i0);
        int mine[kSelLoads], upto[kSelLoads];  // above + equal << 16, of this thread's four slots / of the wave up to them
#pragma unroll
        for (int u = 0; u < kSelLoads; ++u) {
            mine[u] = upto[u] = 0;
            if (i0 + u * 4 * kSelThreads < old) {  // (uniform)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i0 + 4 * tid + u * 4 * kSelThreads + j < old) mine[u] += k[u][j] > prefix ? 1 : k[u][j] == prefix ? 1 << 16 : 0;
                upto[u] = lane_sums(mine[u]);
            }
            if (lane == 63) counts[u * kSelWaves + wave] = int2{upto[u] & 0xFFFF, upto[u] >> 16};
        }
        __syncthreads();
        // the sums before every wave's every load (128 of them, two to a lane)
        const int2 c0 = counts[2 * lane], c1 = counts[2 * lane + 1];
        const int2 ends = {lane_sums(c0.x + c1.x), lane_sums(c0.y + c1.y)};
#pragma unroll
        for (int u = 0; u < kSelLoads; ++u) {
            if (i0 + u * 4 * kSelThreads >= old) break;  // (uniform)
            const int at = u * kSelWaves + wave, holder = at >> 1;
            int a = above + __builtin_amdgcn_readlane(ends.x, holder) - __builtin_amdgcn_readlane(c1.x, holder);
            int e = equal + __builtin_amdgcn_readlane(ends.y, holder) - __builtin_amdgcn_readlane(c1.y, holder);
            if ((at & 1) == 0) {
                a -= __builtin_amdgcn_readlane(c0.x, holder);
                e -= __builtin_amdgcn_readlane(c0.y, holder);
            }
            a += (upto[u] - mine[u]) & 0xFFFF;
            e += (upto[u] - mine[u]) >> 16;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = i0 + 4 * tid + u * 4 * kSelThreads + j;
                const bool over = i < old && k[u][j] > prefix, same = i < old && k[u][j] == prefix;
                if (over || (same && e < want)) out[a + min(e, want)] = i;
                a += over;
                e += same;
            }
        }
        above += __builtin_amdgcn_readlane(ends.x, 63);
        equal += __builtin_amdgcn_readlane(ends.y, 63);
        __syncthreads();  // (the counts are written again)
    }
}

// One wave per (row, head, block of eight kept slots): codes, scales and weights of the chosen slots, to their new places
template <int D>
__global__ __launch_bounds__(256) void kv4_move_kernel(after_kv4 c, after_kv4 to, int keep, const int* slots, int nb, long long items) {
    constexpr int G = D / 32;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long item = (long long)blockIdx.x * 4 + wave;
    if (item >= items) return;
    const int rh = (int)(item / nb), sb = (int)(item % nb), r = rh / c.kv_heads;
    const int n = min(row_length(c, r), keep), m = min(n - 8 * sb, 8);
    if (sb == 0 && lane == 0 && rh % c.kv_heads == 0) to.lengths[r] = n;
    if (m <= 0) return;
    const size_t src = (size_t)rh * c.capacity, dst = (size_t)rh * to.capacity + 8 * sb;
    const int pick = lane < m ? max(slots[(size_t)rh * keep + 8 * sb + lane], 0) : 0;  // (slot 0 for what is not there: read, not used)
    u32x2 x[8];
    if (2 * lane < D) {
#pragma unroll
        for (int tt = 0; tt < 8; ++tt) {
            const int s = __builtin_amdgcn_readlane(pick, tt);
            x[tt] = reinterpret_cast<const u32x2*>(c.values + (src + s) / 8 * (4 * D))[lane];
        }
    }
    // keys: 16 bytes per lane; scales: a token's group per lane
    const int kt = lane / (D / 32), kc = lane % (D / 32), gt = lane / G, g = lane % G;
    u32x4 k;
    unsigned char ks, vs;
    const size_t from = src + __shfl(pick, gt);
    if (lane < 8 * G) {
        k = reinterpret_cast<const u32x4*>(c.keys + (src + __shfl(pick, kt)) * (D / 2))[kc];
        ks = c.key_scales[from * G + g];
        vs = c.value_scales[from * G + g];
    }
    if (lane < m) to.weights[dst + lane] = c.weights[src + pick];
    if (lane < m * G) {
        reinterpret_cast<u32x4*>(to.keys + (dst + kt) * (D / 2))[kc] = k;
        to.key_scales[(dst + gt) * G + g] = ks;
        to.value_scales[(dst + gt) * G + g] = vs;
    }
    if (2 * lane < D) {
        u32x2 y = {0, 0};
#pragma unroll
        for (int tt = 0; tt < 8; ++tt) {
            const int s = __builtin_amdgcn_readlane(pick, tt);
            if (tt < m) y = y | (x[tt] >> 4 * (s & 7) & 15u) << 4 * tt;
        }
        reinterpret_cast<u32x2*>(to.values + dst / 8 * (4 * D))[lane] = y;
    }
}

// ---------------------------------------------------------------------------------------------------------------- host
int check_cache(const after_kv4* c, const char* what) {
    AFTER_REQUIRE(c, AFTER_E_INVALID, "%s: no cache", what);
    AFTER_REQUIRE(c->keys && c->key_scales && c->values && c->value_scales && c->weights && c->lengths && c->failed, AFTER_E_INVALID,
                  "%s: a buffer of the cache is missing", what);
    AFTER_REQUIRE(c->rows > 0 && c->kv_heads > 0 && (c->head_dim == 64 || c->head_dim == 128), AFTER_E_INVALID,
                  "%s: rows and kv_heads > 0, head_dim 64 or 128 (got %d, %d, %d)", what, c->rows, c->kv_heads, c->head_dim);
    AFTER_REQUIRE(c->capacity > 0 && c->capacity % 32 == 0 && c->capacity <= (1 << 24), AFTER_E_INVALID,
                  "%s: capacity a multiple of 32, at most 2^24 (got %d)", what, c->capacity);
    AFTER_REQUIRE((long long)c->rows * c->kv_heads <= (1 << 20), AFTER_E_INVALID, "%s: rows x kv_heads is at most 2^20", what);
    return AFTER_OK;
}
// (a grid's threads are counted in 32 bits: at most 2^24 - 1 workgroups of 256)
constexpr long long kMaxGroups = (1 << 24) - 1;
bool known_type(int t) { return t == AFTER_T_F32 || t == AFTER_T_BF16 || t == AFTER_T_F16; }
int type_bytes(int t) { return t == AFTER_T_F32 ? 4 : 2; }
bool aligned16(const void* p) { return ((size_t)p & 15) == 0; }

struct Plan {
    int m_rows, nm, mgroups;
    int wgs;     // workgroups of four workers, or 0
    int splits;  // of a row, for more than 32 queries; or 0
    long long pieces, o_bytes, ml_bytes, s_bytes, e_bytes, f_bytes;
    long long total() const { return o_bytes + ml_bytes + s_bytes + e_bytes + f_bytes; }
};
// How many columns of a product the queries take: with the others for their pieces, where they fit
constexpr int attend_cols(int type, int m_rows) { return type == AFTER_T_F16 && m_rows <= 8 ? 8 : type == AFTER_T_F32 && m_rows <= 4 ? 4 : 16; }
Plan attend_plan(const after_kv4& c, int type, int heads, int tokens, bool count) {
    Plan p;
    p.m_rows = tokens * (heads / c.kv_heads);
    p.nm = p.m_rows > 16 ? 2 : 1;
    p.mgroups = p.m_rows > 32 ? cdiv(p.m_rows, kWideRows) : 1;
    p.wgs = p.splits = 0;
    const long long n_rh = (long long)c.rows * c.kv_heads, most = cdivll(n_rh * (c.capacity / kStep), 4);
    if (p.m_rows > 32) {
        // two workgroups on each of 256 CUs, and no split below four tiles
        const long long wanted = cdivll(512, n_rh * p.mgroups), tiles = cdivll(c.capacity, 4 * kWideTile);
        p.splits = (int)(wanted < tiles ? wanted : tiles);
    } else if (c.capacity > 512) {
        // Workers for two workgroups on each of 256 CUs, for three where the queries' registers leave room and there are many rows
        // (with few, more pieces are a longer join), for one where two do not fit a CU.  Up to 16 queries of a row and head, D = 128,
        // with the join: 64 rows of 1 .. 8192 x 8 heads, bf16 75.6 us against 78.3 with two, fp16 76.3 / 82.0, fp32 81.4 / 87.2
        // (without pieces in columns 81.7 and 88.2); 8 rows of 1 .. 32767, bf16 45.2 / 45.7; two rows of 131071, bf16 71.6 / 68.4,
        // fp16 72.1 / 69.0; one of 32768 26.9 / 23.6.  24 queries, D = 128, calls one behind the other on the same cache: bf16 (two
        // fit) 8 rows of 1 .. 32767 59.3 us against 67.7 with three, 32 of 1 .. 8192 56.6 / 65.4, 64 of 4096 86.6 / 106.8, but 64 of
        // 1 .. 8192 126.4 / 110.3; fp16 and fp32 (one fits) 8 rows 87.6 and 110.2 against 99.1 and 121.5 with two, 64 rows of
        // 1 .. 8192 181.8 and 209.3 / 185.3 and 214.9.
        // Rows of at most 512 slots take a workgroup each and one launch: 6.2 us against 9.
        const int full = p.nm == 2 ? (type != AFTER_T_BF16 && c.head_dim == 128 ? 256 : 512)
                         : n_rh >= 64 && (attend_cols(type, p.m_rows) < 16 || type == AFTER_T_BF16) ? 768
                                                                                                    : 512;
        p.wgs = (int)(most < full ? most : full);
    }
    p.pieces = p.splits ? n_rh * p.splits : 4ll * p.wgs + n_rh;
    p.o_bytes = p.wgs || p.splits > 1 ? p.pieces * p.m_rows * c.head_dim * 4 : 0;
    p.ml_bytes = p.wgs || p.splits ? (p.pieces * p.m_rows * 8 + 255) / 256 * 256 : 0;
    p.f_bytes = count ? (n_rh * p.m_rows * 8 + 255) / 256 * 256 : 0;
    p.s_bytes = count && !p.splits ? n_rh * p.m_rows * c.capacity * 4 : 0;
    p.e_bytes = p.wgs || p.splits ? (n_rh * 8 + 255) / 256 * 256 : 0;
    return p;
}

template <int TYPE, int D, int NM, bool COUNT, int COLS>
void launch_attend(const AttendArgs& a, const Plan& p, hipStream_t s) {
    constexpr size_t ring = 4 * kRing * kTileBytes<D>, out = 4 * 16 * (D + 4) * 4;  // (at most 53 KB: three workgroups a CU)
    if (p.wgs)
        hipLaunchKernelGGL((kv4_attend_kernel<TYPE, D, NM, COUNT, false, COLS>), dim3(p.wgs), dim3(256), ring, s, a);
    else
        hipLaunchKernelGGL((kv4_attend_kernel<TYPE, D, NM, COUNT, true, COLS>), dim3(a.c.rows * a.c.kv_heads), dim3(256), ring > out ? ring : out, s, a);
}

template <int TYPE, int D>
int run_attend(const AttendArgs& a, const Plan& p, bool count, float decay, hipStream_t s) {
    const int n_rh = a.c.rows * a.c.kv_heads;
    if (p.splits) {
        static LdsAttr attr;
        constexpr size_t lds = 4 * Widen<D>::KEYS;
        AFTER_TRY(ensure_lds_attr(attr, (const void*)kv4_wide_kernel<TYPE, D>, lds));
        const long long grid = cdivll((long long)n_rh * p.splits, 8) * 8 * p.mgroups;
        hipLaunchKernelGGL((kv4_wide_kernel<TYPE, D>), dim3((unsigned)grid), dim3(256), lds, s, a, p.splits, p.mgroups);
        // (empty rows have no workgroup: their zeros come from the join)
        hipLaunchKernelGGL((kv4_join_kernel<TYPE, D>), dim3(n_rh * a.m_rows), dim3(256), 0, s, a);
        if (count) {
            const long long even = cdivll((long long)n_rh * a.c.capacity, 768 * kWideTile) * kWideTile;  // three workgroups a CU
            const int slots = (int)(even < 256 ? 256 : even < kWideSlots ? even : kWideSlots), blocks = cdiv(a.c.capacity, slots);
            hipLaunchKernelGGL((kv4_wide_weights_kernel<TYPE, D>), dim3((unsigned)(n_rh * blocks)), dim3(256), 2 * Widen<D>::KEYS, s, a, blocks, slots, decay);
        }
        AFTER_HIP_CHECK(hipGetLastError());
        return AFTER_OK;
    }
    constexpr int few = attend_cols(TYPE, 1);
    if (few < 16 && attend_cols(TYPE, p.m_rows) == few) {
        if (count)
            launch_attend<TYPE, D, 1, true, few>(a, p, s);
        else
            launch_attend<TYPE, D, 1, false, few>(a, p, s);
    } else if (p.nm == 1) {
        if (count)
            launch_attend<TYPE, D, 1, true, 16>(a, p, s);
        else
            launch_attend<TYPE, D, 1, false, 16>(a, p, s);
    } else {
        if (count)
            launch_attend<TYPE, D, 2, true, 16>(a, p, s);
        else
            launch_attend<TYPE, D, 2, false, 16>(a, p, s);
    }
    if (p.wgs)
        hipLaunchKernelGGL((kv4_join_kernel<TYPE, D>), dim3(n_rh * a.m_rows), dim3(256), 0, s, a);
    if (count) {
        const int slots = cdiv(a.c.capacity, 1024);
        hipLaunchKernelGGL(kv4_weights_kernel, dim3(n_rh * slots), dim3(256), 0, s, a, slots, decay);
    }
    AFTER_HIP_CHECK(hipGetLastError());
    return AFTER_OK;
}

#define KV4_BY_TYPE(type, dim, CALL)                                       \
    do {                                                                   \
        if ((dim) == 64) {                                                 \
            if ((type) == AFTER_T_F32) CALL(AFTER_T_F32, 64);              \
            else if ((type) == AFTER_T_BF16) CALL(AFTER_T_BF16, 64);       \
            else CALL(AFTER_T_F16, 64);                                    \
        } else {                                                           \
            if ((type) == AFTER_T_F32) CALL(AFTER_T_F32, 128);             \
            else if ((type) == AFTER_T_BF16) CALL(AFTER_T_BF16, 128);      \
            else CALL(AFTER_T_F16, 128);                                   \
        }                                                                  \
    } while (0)

}  // namespace
}  // namespace after

using namespace after;

extern "C" int after_kv4_append(const after_kv4* c, const void* k, const void* v, int type, const int* starts, int tokens, long long total,
                                long long k_token_stride, long long k_head_stride, long long v_token_stride, long long v_head_stride, void* stream) {
    AFTER_TRY(check_cache(c, "kv4_append"));
    AFTER_REQUIRE(known_type(type), AFTER_E_INVALID, "kv4_append: unknown element type %d", type);
    AFTER_REQUIRE(total >= 0 && total < (1ll << 30) && tokens >= 0, AFTER_E_INVALID, "kv4_append: 0 <= total < 2^30 new tokens (got %lld)", total);
    AFTER_REQUIRE(starts || (long long)tokens * c->rows == total, AFTER_E_INVALID, "kv4_append: total = rows x tokens without starts");
    if (total == 0) return AFTER_OK;
    const int per16 = 16 / type_bytes(type);
    AFTER_REQUIRE(k && v && aligned16(k) && aligned16(v) && k_token_stride % per16 == 0 && k_head_stride % per16 == 0 && v_token_stride % per16 == 0 &&
                      v_head_stride % per16 == 0,
                  AFTER_E_INVALID, "kv4_append: k and v, their token and head strides must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    const NewTokens nt{starts, tokens, (int)total};
    const long long items = (total / 8 + 2ll * c->rows) * c->kv_heads;
    AFTER_REQUIRE(cdivll(items, 4) <= kMaxGroups, AFTER_E_INVALID, "kv4_append: too many new tokens x heads for one call");
    const AppendArgs a{*c, nt, k, v, k_token_stride, k_head_stride, v_token_stride, v_head_stride};
    // A workgroup per row where no row can have many: 64 rows of one token each in one launch.  (`starts` may give all to one row.)
    if (starts ? total <= 2ll * c->rows && total <= 256 : tokens <= 16) {
#define CALL(T, D) hipLaunchKernelGGL((kv4_append_rows_kernel<T, D>), dim3(c->rows), dim3(512), 0, s, a)
        KV4_BY_TYPE(type, c->head_dim, CALL);
#undef CALL
    } else {
#define CALL(T, D) hipLaunchKernelGGL((kv4_append_kernel<T, D>), dim3((unsigned)cdivll(items, 4)), dim3(256), 0, s, a, (int)items)
        KV4_BY_TYPE(type, c->head_dim, CALL);
#undef CALL
        hipLaunchKernelGGL(kv4_advance_kernel, dim3(cdiv(c->rows, 256)), dim3(256), 0, s, *c, nt);
    }
    AFTER_HIP_CHECK(hipGetLastError());
    return AFTER_OK;
}

extern "C" int after_kv4_truncate(const after_kv4* c, const int* lengths, void* stream) {
    AFTER_TRY(check_cache(c, "kv4_truncate"));
    hipLaunchKernelGGL(kv4_truncate_kernel, dim3(cdiv(c->rows, 256)), dim3(256), 0, (hipStream_t)stream, *c, lengths);
    AFTER_HIP_CHECK(hipGetLastError());
    return AFTER_OK;
}

extern "C" int after_kv4_read(const after_kv4* c, void* k, void* v, int type, const int* start, int count, void* stream) {
    AFTER_TRY(check_cache(c, "kv4_read"));
    AFTER_REQUIRE(type == AFTER_T_F32 || type == AFTER_T_BF16, AFTER_E_INVALID, "kv4_read: values are written as fp32 or bf16 (both hold them exactly)");
    AFTER_REQUIRE(count >= 0 && count <= c->capacity, AFTER_E_INVALID, "kv4_read: 0 <= count <= capacity (got %d)", count);
    if (count == 0) return AFTER_OK;
    AFTER_REQUIRE(k && v && aligned16(k) && aligned16(v), AFTER_E_INVALID, "kv4_read: k and v must be 16-byte aligned");
    const int nb = count / 8 + 2;
    const long long items = (long long)c->rows * c->kv_heads * nb;
    AFTER_REQUIRE(cdivll(items, 4) <= kMaxGroups, AFTER_E_INVALID, "kv4_read: too many slots x heads for one call");
#define CALL(T, D) \
    hipLaunchKernelGGL((kv4_read_kernel<T, D>), dim3((unsigned)cdivll(items, 4)), dim3(256), 0, (hipStream_t)stream, *c, k, v, start, count, nb, items)
    if (c->head_dim == 64) {
        if (type == AFTER_T_F32) CALL(AFTER_T_F32, 64);
        else CALL(AFTER_T_BF16, 64);
    } else {
        if (type == AFTER_T_F32) CALL(AFTER_T_F32, 128);
        else CALL(AFTER_T_BF16, 128);
    }
#undef CALL
    AFTER_HIP_CHECK(hipGetLastError());
    return AFTER_OK;
}

static int check_attend(const after_kv4* c, int type, int heads, int tokens, const char* what) {
    AFTER_TRY(check_cache(c, what));
    AFTER_REQUIRE(known_type(type), AFTER_E_INVALID, "%s: unknown element type %d", what, type);
    AFTER_REQUIRE(heads > 0 && heads % c->kv_heads == 0, AFTER_E_INVALID, "%s: heads must be a multiple of the cache's %d", what, c->kv_heads);
    AFTER_REQUIRE(tokens > 0 && (long long)tokens * (heads / c->kv_heads) <= 65536, AFTER_E_INVALID, "%s: 1 .. 65536 / (heads / kv_heads) tokens (got %d)",
                  what, tokens);
    const Plan p = attend_plan(*c, type, heads, tokens, false);
    const long long n_rh = (long long)c->rows * c->kv_heads;
    AFTER_REQUIRE((p.splits ? n_rh * p.splits + 8 : n_rh) * p.mgroups <= kMaxGroups && n_rh * p.m_rows <= kMaxGroups &&
                      n_rh * cdiv(c->capacity, 256) <= kMaxGroups,
                  AFTER_E_INVALID, "%s: too many rows x heads x tokens for one call", what);
    return AFTER_OK;
}

extern "C" int after_kv4_attend_workspace(const after_kv4* c, int type, int heads, int tokens, int accumulate, long long* bytes) {
    AFTER_TRY(check_attend(c, type, heads, tokens, "kv4_attend_workspace"));
    AFTER_REQUIRE(bytes, AFTER_E_INVALID, "kv4_attend_workspace: bytes is NULL");
    const Plan p = attend_plan(*c, type, heads, tokens, accumulate != 0);
    *bytes = p.total();
    return AFTER_OK;
}

extern "C" int after_kv4_attend(const after_kv4* c, const after_kv4_query* query, void* stream) {
    AFTER_REQUIRE(query, AFTER_E_INVALID, "kv4_attend: no query");
    const after_kv4_query& x = *query;
    AFTER_TRY(check_attend(c, x.type, x.heads, x.tokens, "kv4_attend"));
    const int per16 = 16 / type_bytes(x.type);
    AFTER_REQUIRE(x.q && x.out && aligned16(x.q) && aligned16(x.out) && x.q_row_stride % per16 == 0 && x.q_token_stride % per16 == 0 && x.q_head_stride % per16 == 0,
                  AFTER_E_INVALID, "kv4_attend: q, its strides and out must be 16-byte aligned");
    AFTER_REQUIRE(std::isfinite(scale_log2(x.scale)) && !std::isnan(x.scale) && std::isfinite(x.decay), AFTER_E_INVALID,
                  "kv4_attend: scale (times log2 e too) and decay must be finite");
    const bool count = x.accumulate != 0;
    const Plan p = attend_plan(*c, x.type, x.heads, x.tokens, count);
    const long long need = p.total();
    AFTER_REQUIRE(need == 0 || (x.workspace && aligned16(x.workspace) && x.workspace_bytes >= need), AFTER_E_CAPACITY,
                  "kv4_attend: needs a 16-byte aligned workspace of %lld bytes (got %lld)", need, x.workspace_bytes);
    AttendArgs a;
    a.c = *c;
    a.q = x.q;
    a.out = x.out;
    a.qrs = x.q_row_stride;
    a.qts = x.q_token_stride;
    a.qhs = x.q_head_stride;
    a.heads = x.heads;
    a.tokens = x.tokens;
    a.group = x.heads / c->kv_heads;
    a.m_rows = p.m_rows;
    a.workers = 4 * p.wgs;
    a.pieces = (int)p.pieces;
    a.scale2 = scale_log2(x.scale);
    a.q_sign = x.scale < 0 ? -1.f : 1.f;
    char* w = (char*)x.workspace;
    a.scores = (float*)w;
    a.part_ml = (f32x2*)(w += p.s_bytes);
    a.final_ml = count ? (f32x2*)(w + p.ml_bytes) : nullptr;
    a.ends = (int2*)(w += p.ml_bytes + p.f_bytes);
    a.part_o = (float*)(w += p.e_bytes);
#define CALL(T, D) return run_attend<T, D>(a, p, count, x.decay, (hipStream_t)stream)
    KV4_BY_TYPE(x.type, c->head_dim, CALL);
#undef CALL
    return AFTER_OK;
}

extern "C" int after_kv4_evict(const after_kv4* c, const after_kv4* to, int keep, int recent, int* slots, void* stream) {
    AFTER_TRY(check_cache(c, "kv4_evict"));
    AFTER_TRY(check_cache(to, "kv4_evict"));
    AFTER_REQUIRE(to->rows == c->rows && to->kv_heads == c->kv_heads && to->head_dim == c->head_dim, AFTER_E_INVALID,
                  "kv4_evict: both caches need the same rows, kv_heads and head_dim");
    AFTER_REQUIRE(to->keys != c->keys && to->lengths != c->lengths, AFTER_E_INVALID, "kv4_evict: the slots move into another cache");
    AFTER_REQUIRE(keep > 0 && keep <= to->capacity, AFTER_E_CAPACITY, "kv4_evict: keep %d slots, the other cache holds %d", keep, to->capacity);
    AFTER_REQUIRE(recent >= 0 && recent <= keep, AFTER_E_INVALID, "kv4_evict: 0 <= recent <= keep (got %d of %d)", recent, keep);
    AFTER_REQUIRE(slots, AFTER_E_INVALID, "kv4_evict: slots is NULL");
    hipStream_t s = (hipStream_t)stream;
    const int n_rh = c->rows * c->kv_heads, nb = cdiv(keep, 8);
    const long long items = (long long)n_rh * nb;
    AFTER_REQUIRE(cdivll(items, 4) <= kMaxGroups && n_rh <= kMaxGroups / 4, AFTER_E_INVALID, "kv4_evict: too many slots x heads for one call");
    hipLaunchKernelGGL(kv4_select_kernel, dim3(n_rh), dim3(kSelThreads), 0, s, *c, keep, recent, slots);
    if (c->head_dim == 64)
        hipLaunchKernelGGL((kv4_move_kernel<64>), dim3((unsigned)cdivll(items, 4)), dim3(256), 0, s, *c, *to, keep, slots, nb, items);
    else
        hipLaunchKernelGGL((kv4_move_kernel<128>), dim3((unsigned)cdivll(items, 4)), dim3(256), 0, s, *c, *to, keep, slots, nb, items);
    AFTER_HIP_CHECK(hipGetLastError());
    return AFTER_OK;
}
