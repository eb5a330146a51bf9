// Attention of packed sequences (include/after_hip.h: after_attend_packed; Python: after_amd.attend_packed).
//
// Mathematics.  One pass over the keys with the running maximum m and sum l of the softmax: a tile's scores s raise m to m',
// what is summed so far shrinks by 2^(m - m'), p = 2^(s - m') (scores carry log2 e).  Scores and output are formed transposed,
// S^T = K Q^T and O^T = V^T P^T, so that a query is a lane: its maximum and sum are a chain over the lane's registers and one
// exchange with the other half of the wave, and a rescale is one factor per lane.  Row i of a 32 x 32 result stands at
// 8 (i / 4) + 4 (lane / 32) + i % 4; with the contraction of the second product taken in that same order, the probabilities
// are its operand as they lie, and only V is read accordingly (two transposing LDS reads per 16 tokens).
//
// Rows.  The `group` heads that share a key head are rows of one tile, row = token * group + head: short sequences fill tiles,
// and a key tile is read once for all of them.  A workgroup holds 128 rows, 32 to a wave (or 32 in all: "few rows" below); its
// tile number alone says which sequence it serves (sequence b owns the numbers from floor(start_b * group / 128) + b on), so the
// grid needs no lengths.
//
// What bounds it.  Long prompts: the matrix pipes, with the softmax's exponentials between two products; 16384 causal tokens, bf16,
// 32 / 8 heads of 128: 2070 .. 2200 us from card to card, 1000 .. 1060 TFLOP/s, where a large product of the library reaches 1155
// (fp16 heads of 128 in a batch of 1 .. 2047 tokens: 297 .. 312 us, 700 .. 735, its workgroups' beginnings and ends stand alone; heads
// of 64, 8192 tokens: 313 us, 880; fp32 heads of 128, 4096 tokens: 580 us, 118 of 153).
// Tiles of 64 keys, two of them in LDS and two workgroups on a CU: one computes while the other waits.  Measured and left out:
// V read by instructions that wait by themselves, and scheduling hints (the same time), skipping the unseen half of a masked
// tile (2330 us).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "attention.h"
#include "common.h"
#include "gemm_pipe.h"

namespace after {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int BM = 128, BN = 64;
// In fp16 products probabilities, and the sum that divides them, are held 2^7 times as large: up to 2^15 with a maximum that moves at
// 2^8, and what is rounded to nothing is below 2^-32 of the largest, where without it keys 25.2 octaves below vanished from the
// output but not from the sum (2^17 of them and a key of value 0: 0 instead of 0.0034).
template <int TYPE>
constexpr float kLift = TYPE == AFTER_T_F16 ? 7.f : 0.f;

template <int TYPE>
struct Elem;
template <>
struct Elem<AFTER_T_F32> {
    using T = float;
};
template <>
struct Elem<AFTER_T_BF16> {
    using T = __bf16;
    using V8 = bf16x8;
    static __device__ __forceinline__ f32x16 mfma(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Elem<AFTER_T_F16> {
    using T = _Float16;
    using V8 = f16x8;
    static __device__ __forceinline__ f32x16 mfma(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// n / d for 0 <= n < 2^31 by a product (d is the same for all: found on the host)
struct Divisor {
    unsigned d, magic, shift;
    __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi((unsigned)n, magic) + (unsigned)n) >> shift); }
};
Divisor divisor(unsigned d) {
    unsigned shift = 0;
    while ((1ull << shift) < d) ++shift;
    return Divisor{d, (unsigned)((((1ull << shift) - d) << 32) / d + 1), shift};
}

struct PackedArgs {
    const void *q, *k, *v;
    void* out;
    const int *qs, *ks;
    long long qts, qhs, kts, khs, vts, vhs, ots, ohs;
    int q_rows, k_rows, n_seqs, kv_heads, group, tiles, splits;
    Divisor by_group, by_chunk, by_kv_heads, by_splits;
    float scale2;     // |scale| log2 e, > 0 (a masked score, -inf, stays -inf)
    unsigned q_sign;  // the sign bits of a word of q, if scale is negative
    int causal, window, zero_rest;
    float* part_o;    // [tiles][kv_heads][splits][kFewRows][D], if splits > 1
    f32x2* part_ml;   // the same rows' maxima and sums
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }

// Sequence b of the queries begins at row ...; one more "sequence" without keys stands for the rows behind the last
__device__ __forceinline__ int q_start(const PackedArgs& a, int b) {
    const int x = a.qs[min(b, a.n_seqs)];
    return b <= 0 ? 0 : b > a.n_seqs ? a.q_rows : clampi(x, 0, a.q_rows);
}
__device__ __forceinline__ int k_start(const PackedArgs& a, int b) {
    const int x = a.ks[min(b, a.n_seqs)];
    return b <= 0 ? 0 : clampi(x, 0, a.k_rows);
}

// [first, last) of the keys that the query at position p of its sequence sees (a query older than the keys: p < 0, none)
__device__ __forceinline__ void seen(const PackedArgs& a, int p, int keys, int& first, int& last) {
    first = 0;
    last = keys;
    if (a.causal) {
        const int chunk = (int)a.by_chunk.d, begin = a.by_chunk(max(p, 0)) * chunk;
        last = p < 0 ? 0 : min(begin + chunk, keys);
        if (a.window > 0) first = max(0, min(begin, p - a.window + 1));
    }
}

// Which sequence a tile of ROWS rows serves, and where in it: rows [row0, row0 + ROWS) of the sequence's nq * group; false: none
struct Place {
    int b, q0, nq, k0, nk, row0, rows;
};
template <int ROWS>
__device__ __forceinline__ bool find_tile(const PackedArgs& a, int tile, Place& p) {
    const int lane = threadIdx.x & 63;
    // the last sequence that begins at or before this tile: 64 candidates at a time; the last look holds its ends
    int lo = 0, hi = a.n_seqs, q1, k1;
    for (;;) {
        const int step = (hi - lo + 64) >> 6, at = lo + lane * step, qs = q_start(a, at), ks = k_start(a, at);
        const bool begun = (int)((long long)qs * a.group / ROWS) + at <= tile;
        const int j = 63 - __clzll(__ballot(begun && at <= hi) | 1);  // (sequence lo has begun)
        if (step == 1) {
            p.b = lo + j;
            p.q0 = __builtin_amdgcn_readlane(qs, j);
            p.k0 = __builtin_amdgcn_readlane(ks, j);
            q1 = j < 63 ? __builtin_amdgcn_readlane(qs, (j + 1) & 63) : q_start(a, p.b + 1);
            k1 = j < 63 ? __builtin_amdgcn_readlane(ks, (j + 1) & 63) : k_start(a, p.b + 1);
            break;
        }
        lo += j * step;
        hi = min(hi, lo + step - 1);
    }
    p.nq = q1 - p.q0;
    p.row0 = (tile - ((int)((long long)p.q0 * a.group / ROWS) + p.b)) * ROWS;
    p.rows = p.nq * a.group;  // (< 2^31: checked on the host)
    p.nk = p.b < a.n_seqs ? max(k1 - p.k0, 0) : 0;
    return p.row0 >= 0 && p.row0 < p.rows && (p.b < a.n_seqs || a.zero_rest);
}

// 16-byte pieces of a 64-row tile in LDS.  Keys: a wave reads the same piece of 32 rows, so a row's pieces are permuted by its
// number; values (16-bit types): a transposing read takes 32 bytes each of four neighbouring rows, so pairs of pieces are.
template <int PIECES>
__device__ __forceinline__ int k_flip(int row) {
    return row & (PIECES == 16 ? 15 : 7);
}
template <int PIECES>
__device__ __forceinline__ int v_flip(int row) {
    return (row & (PIECES < 16 ? 3 : 7)) << 1;
}

// whether one of the words' elements is an infinity or NaN
template <int TYPE>
__device__ __forceinline__ bool odd_value(u32x4 w) {
    constexpr unsigned e = TYPE == AFTER_T_F16 ? 0x7C00u : 0x7F80u;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (TYPE == AFTER_T_F32)
            bad |= (w[i] & 0x7F800000u) == 0x7F800000u;
        else
            bad |= (w[i] & e) == e || (w[i] >> 16 & e) == e;
    }
    return bad;
}

// a barrier for what is in LDS: loads on their way stay on their way (__syncthreads waits for them)
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int TYPE, int D>
__global__ __launch_bounds__(256, sizeof(typename Elem<TYPE>::T) * D > 256 ? 1 : 2) void attend_packed_kernel(PackedArgs a) {
    using E = Elem<TYPE>;
    using T = typename E::T;
    constexpr int PIECES = D * (int)sizeof(T) / 16;  // 16-byte pieces of a row
    constexpr int LOADS = BN * PIECES / 256;         // pieces per thread of a tile
    constexpr int DT = D / 32;
    constexpr unsigned STAGE = 2 * BN * PIECES * 16;
    extern __shared__ __align__(16) char lds[];
    __shared__ unsigned long long odd_rows[3];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, half = lane >> 5;
    // neighbouring workgroups are dispatched to different XCDs: a key head's workgroups stay on one L2 where there are eight.
    // Tiles from the last to the first: with a causal mask the longest first.
    const int back = a.by_kv_heads(blockIdx.x), h = blockIdx.x - back * a.kv_heads, tile = a.tiles - 1 - back;
    Place place;
    if (!find_tile<BM>(a, tile, place)) return;
    const int q0 = place.q0, nq = place.nq, k0 = place.k0, nk = place.nk, row0 = place.row0, rows = place.rows;

    // this lane's query, and the keys that its workgroup sees: asked for before the rest is worked out
    const int row = row0 + wave * 32 + l31, t = a.by_group(min(row, rows - 1)), g = min(row, rows - 1) - t * a.group;
    const T* qp = (const T*)a.q + (long long)(q0 + t) * a.qts + (long long)(h * a.group + g) * a.qhs;
    // Q: 16-bit types: step s contracts channels 16 s + 8 half + 0 .. 7; fp32: step s, e channels 8 s + 4 half + e
    constexpr int QN = sizeof(T) == 4 ? D / 8 : D / 16;
    u32x4 qf[QN];
#pragma unroll
    for (int s = 0; s < QN; ++s) qf[s] = *reinterpret_cast<const u32x4*>(qp + (2 * s + half) * (16 / (int)sizeof(T))) ^ a.q_sign;

    int t_first, t_last, dummy;
    seen(a, a.by_group(row0) + nk - nq, nk, t_first, dummy);
    seen(a, a.by_group(min(row0 + BM, rows) - 1) + nk - nq, nk, dummy, t_last);
    const T* kp = (const T*)a.k + (long long)k0 * a.kts + (long long)h * a.khs;
    const T* vp = (const T*)a.v + (long long)k0 * a.vts + (long long)h * a.vhs;

    // K and V tiles go from memory to LDS without passing registers, two stages: while a tile is computed the next is on its way.
    // A lane's place in LDS is its number, so the pieces are permuted by the address it reads from.  Rows behind the sequence
    // repeat its last one: they are masked, and taken out below where that one holds an infinity or NaN.
    const int n_first = t_first / BN, n_last = (t_last + BN - 1) / BN;  // key tiles
    const unsigned lds0 = (unsigned)(unsigned long)(__attribute__((address_space(3))) char*)lds;
    constexpr int ROWS = 256 / PIECES;  // rows that one piece per thread covers: the permutations repeat after them
    const int fr = tid / PIECES, fc = tid % PIECES;
    const unsigned kc = (fc ^ k_flip<PIECES>(fr)) * 16, vc = (sizeof(T) == 4 ? fc : fc ^ v_flip<PIECES>(fr)) * 16;
    const unsigned kb = (unsigned)a.kts * (unsigned)sizeof(T), vb = (unsigned)a.vts * (unsigned)sizeof(T);  // (< 2^24: checked on the host)
    const unsigned k_at = fr * kb + kc, v_at = fr * vb + vc;
    auto fetch = [&](int n, int stage) {
        const unsigned to = lds0 + stage * STAGE + wave * 1024;
        const unsigned long long kt = reinterpret_cast<unsigned long long>(kp) + (unsigned long long)n * BN * kb;
        const unsigned long long vt = reinterpret_cast<unsigned long long>(vp) + (unsigned long long)n * BN * vb;
        if ((n + 1) * BN <= nk) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                lds_dma16(to + i * 4096, k_at, kt + i * ROWS * kb);
                lds_dma16(to + i * 4096 + STAGE / 2, v_at, vt + i * ROWS * vb);
            }
        } else {
            const int left = nk - 1 - n * BN;
            for (int i = 0; i < LOADS; ++i) {
                const unsigned j = min(i * ROWS + fr, left);
                lds_dma16(to + i * 4096, j * kb + kc, kt);
                lds_dma16(to + i * 4096 + STAGE / 2, j * vb + vc, vt);
            }
        }
    };
    if (n_first < n_last) fetch(n_first, 0);
    // the keys that the query sees
    int first, last;
    seen(a, t + nk - nq, nk, first, last);
    // the keys that some query of the wave sees
    int w_first = 0, w_last = 0;
    const int w_row = __builtin_amdgcn_readfirstlane(row0 + wave * 32);
    if (w_row < rows) {
        seen(a, a.by_group(w_row) + nk - nq, nk, w_first, dummy);
        seen(a, a.by_group(min(w_row + 32, rows) - 1) + nk - nq, nk, dummy, w_last);
    }
    // every query of the workgroup sees [all_first, all_last)
    int all_first, all_last;
    seen(a, a.by_group(row0) + nk - nq, nk, dummy, all_last);
    seen(a, a.by_group(min(row0 + BM, rows) - 1) + nk - nq, nk, all_first, dummy);

    f32x16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    float mx = -INFINITY, l = 0.f;
    bool far = false;                                      // some query's maximum is beyond kFarTop
    float off = -kLift<TYPE>, times = a.scale2, limit = -INFINITY;  // p = 2^(score times - off); the maximum moves beyond the limit

    int checked = 0;
    if (tid < 3) odd_rows[tid] = 0;
    for (int n = n_first; n < n_last; ++n) {
        const bool masked = n * BN < all_first || (n + 1) * BN > all_last;
        const int stage = (n - n_first) & 1;
        u32x4* lk = reinterpret_cast<u32x4*>(lds + stage * STAGE);
        u32x4* lv = lk + BN * PIECES;
        wait_vmcnt_imm<0>();
        __syncthreads();  // the tile is there, and nobody reads the other stage any more
        if (n + 1 < n_last) fetch(n + 1, stage ^ 1);
        unsigned long long odd = 0;
        if (masked) {  // what a query does not see must not reach it, but 0 x NaN would
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                if (odd_value<TYPE>(lv[i * 256 + tid])) atomicOr(&odd_rows[checked], 1ull << (i * 256 + tid) / PIECES);
            lds_barrier();
            odd = odd_rows[checked];
            if (odd) {  // (rare) such rows are taken out of the product and added one by one below
#pragma unroll
                for (int i = 0; i < LOADS; ++i)
                    if (odd >> (i * 256 + tid) / PIECES & 1) lv[i * 256 + tid] = u32x4{0, 0, 0, 0};
                lds_barrier();
            }
            // (three words in turn: this one has been read by all before the next barrier, and is written again two barriers on)
            checked = checked == 2 ? 0 : checked + 1;
            if (tid == 0) odd_rows[checked == 2 ? 0 : checked + 1] = 0;
        }

        if (masked && (n * BN >= w_last || (n + 1) * BN <= w_first)) continue;  // (nothing in it that this wave sees)
        f32x16 sc[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[f][e] = 0.f;
#pragma unroll
            for (int s = 0; s < QN; ++s) {
                const u32x4 kf = lk[(32 * f + l31) * PIECES + ((2 * s + half) ^ k_flip<PIECES>(l31))];
                if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sc[f] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(kf[e]), __uint_as_float(qf[s][e]), sc[f], 0, 0, 0);
                } else
                    sc[f] = E::mfma(__builtin_bit_cast(typename E::V8, kf), __builtin_bit_cast(typename E::V8, qf[s]), sc[f]);
            }
        }
        if (masked) {
            const int j0 = n * BN + 4 * half;
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int j = j0 + 32 * f + 8 * (e >> 2) + (e & 3);
                    sc[f][e] = j >= first && j < last ? sc[f][e] : -INFINITY;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, sc[f][e]);
        top = fmaxf(top, __shfl_xor(top, 32)) * a.scale2;
        // the maximum moves only when scores outgrow it by 2^8: probabilities up to 256 are as exact, and a rescale is rare
        // (where the maximum is beyond kFarTop, scores are brought down here in every tile: the usual one has no branch for it)
        if (__any(top > limit)) {
            const float now = fmaxf(mx, top), f = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx - now);
            mx = now;
            far = __any(fabsf(now) > kFarTop && now != -INFINITY);
            off = (far || now == -INFINITY ? 0.f : now) - kLift<TYPE>, times = far ? 1.f : a.scale2, limit = far ? -INFINITY : now + 8.f;
            l *= f;
#pragma unroll
            for (int i = 0; i < DT; ++i) o[i] = o[i] * f;
            if (far) {
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sc[g][e] = scaled_below(sc[g][e], a.scale2, mx == -INFINITY ? 0.f : mx);
            }
        }
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                sc[f][e] = __builtin_amdgcn_exp2f(fmaf(sc[f][e], times, -off));
                l += sc[f][e];
            }
        // O^T += V^T P^T
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            if constexpr (sizeof(T) == 4) {
                const float* vv = reinterpret_cast<const float*>(lv);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int j = 32 * f + 8 * (e >> 2) + 4 * half + (e & 3);
#pragma unroll
                    for (int i = 0; i < DT; ++i) o[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(vv[j * D + 32 * i + l31], sc[f][e], o[i], 0, 0, 0);
                }
            } else {
                const char* vv = reinterpret_cast<const char*>(lv);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    typename E::V8 pf;
#pragma unroll
                    for (int e = 0; e < 8; ++e) pf[e] = (T)sc[f][8 * s + e];  // (the products' own type: half a step, 2^-8 / 2^-11, each)
#pragma unroll
                    for (int i = 0; i < DT; ++i) {
                        // lane l of 16 reads 8 bytes of row l / 4: it gets column l of the four rows
                        union {
                            typename E::V8 v;
                            s16x4 p[2];
                        } vf;
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            const int r = 32 * f + 16 * s + 8 * w + 4 * half + ((lane & 15) >> 2);
                            const int byte = 64 * i + (lane & 16) * 2 + (lane & 3) * 8;
                            vf.p[w] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                (__attribute__((address_space(3))) s16x4*)(vv + 16 * (r * PIECES + ((byte >> 4) ^ v_flip<PIECES>(r))) + (byte & 15)));
                        }
                        o[i] = E::mfma(vf.v, pf, o[i]);
                    }
                }
            }
        }
        while (odd) {  // (uniform) rows of V with infinities or NaN in a masked tile: only for the queries that see them
            const int j = __ffsll((unsigned long long)odd) - 1, at = n * BN + j;
            odd &= odd - 1;
            const int e_at = (j >> 3 & 3) * 4 + (j & 3), holder = (j >> 2 & 1) * 32 + l31;
            float p = 0.f;
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if ((j >> 5) == f && e == e_at) p = sc[f][e];
            p = __shfl(p, holder);
            if (at >= first && at < last) {
#pragma unroll
                for (int i = 0; i < DT; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        o[i][e] = fmaf(p, (float)vp[(long long)at * a.vts + 32 * i + 8 * (e >> 2) + 4 * half + (e & 3)], o[i][e]);
            }
        }
    }

    // to memory by way of LDS: a lane holds one row's every eighth group of four channels, a store of whole rows takes half the time
    l += __shfl_xor(l, 32);
    const float inv = inverse_sum(l, first < last);
    constexpr int PITCH = D * (int)sizeof(T) + 16;
    char* mine = lds + wave * (32 * PITCH);
    lds_barrier();  // (the tiles are no longer read)
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            typedef T T4 __attribute__((ext_vector_type(4)));
            T4 y;
#pragma unroll
            for (int w = 0; w < 4; ++w) y[w] = (T)(o[i][e + w] * inv);
            *reinterpret_cast<T4*>(mine + l31 * PITCH + (32 * i + 2 * e + 4 * half) * sizeof(T)) = y;
        }
#pragma unroll
    for (int i = 0; i < 32 * PIECES / 64; ++i) {
        const int id = i * 64 + lane, r = id / PIECES, c = id % PIECES, at = row0 + wave * 32 + r;
        if (at < rows) {
            const int tr = a.by_group(at), gr = at - tr * a.group;
            *reinterpret_cast<u32x4*>((T*)a.out + (long long)(q0 + tr) * a.ots + (long long)(h * a.group + gr) * a.ohs + c * (16 / (int)sizeof(T))) =
                *reinterpret_cast<const u32x4*>(mine + r * PITCH + c * 16);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------- few rows
// Where tiles of 128 rows would leave most of the chip idle (short prompts, a few new tokens over many keys): 32 rows to a
// workgroup, whose four waves share out their keys, 32 at a time.  Each wave has one buffer for keys and one for values in LDS:
// the next keys are asked for when the scores are formed, the next values when they are added up, and no wave waits for another
// until the four are joined.  With `splits` > 1 that many workgroups share the keys, and attend_join_kernel joins them.
// What bounds it: short sequences, the chain of loads before the first product (3 x 256 fp32 tokens of 8 heads of 64, window 8: 8.6
// us); one query over many keys, memory (bf16, 8 heads of 128: 32768 keys 28.4 us, 131072 102 us = 5.2 TB/s).
constexpr int kFewRows = 32;
// steps of 32 keys per wave, and the workgroups that have any
__device__ __forceinline__ int few_share(const PackedArgs& a, int steps) { return max(1, (steps + 4 * a.splits - 1) / (4 * a.splits)); }
__device__ __forceinline__ int few_used(int steps, int share) { return (steps + 4 * share - 1) / (4 * share); }
// the keys that some / every query of the tile sees
__device__ __forceinline__ void few_seen(const PackedArgs& a, const Place& p, int& t_first, int& t_last, int& all_first, int& all_last) {
    const int p0 = p.nk - p.nq;
    seen(a, a.by_group(p.row0) + p0, p.nk, t_first, all_last);
    seen(a, a.by_group(min(p.row0 + kFewRows, p.rows) - 1) + p0, p.nk, all_first, t_last);
}

template <int TYPE, int D>
__global__ __launch_bounds__(256, sizeof(typename Elem<TYPE>::T) * D > 256 ? 1 : 2) void attend_few_kernel(PackedArgs a) {
    using E = Elem<TYPE>;
    using T = typename E::T;
    constexpr int PIECES = D * (int)sizeof(T) / 16, LOADS = PIECES / 2, DT = D / 32;
    constexpr int RW = 64 / PIECES;                // rows that one piece per lane covers
    constexpr unsigned HALF = kFewRows * D * sizeof(T);  // bytes of 32 keys
    extern __shared__ __align__(16) char lds[];    // [4][keys, values]; then [4][32][D + 4] floats

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, half = lane >> 5;
    const int back = a.by_kv_heads(blockIdx.x), h = blockIdx.x - back * a.kv_heads, of = a.by_splits(back), split = back - of * a.splits;
    const int tile = a.tiles - 1 - of;
    Place place;
    if (!find_tile<kFewRows>(a, tile, place)) return;
    const int q0 = place.q0, nq = place.nq, nk = place.nk, row0 = place.row0, rows = place.rows;
    int t_first, t_last, all_first, all_last;
    few_seen(a, place, t_first, t_last, all_first, all_last);
    const int steps = (max(t_last - t_first, 0) + 31) / 32, share = few_share(a, steps), used = few_used(steps, share);
    if (split > 0 && split >= used) return;
    const int begin = min((split * 4 + wave) * share, steps), end = min(begin + share, steps);

    const int row = min(row0 + l31, rows - 1), t = a.by_group(row), g = row - t * a.group;
    int first, last;
    seen(a, t + nk - nq, nk, first, last);
    const T* qp = (const T*)a.q + (long long)(q0 + t) * a.qts + (long long)(h * a.group + g) * a.qhs;
    const T* kp = (const T*)a.k + (long long)place.k0 * a.kts + (long long)h * a.khs;
    const T* vp = (const T*)a.v + (long long)place.k0 * a.vts + (long long)h * a.vhs;
    constexpr int QN = sizeof(T) == 4 ? D / 8 : D / 16;
    u32x4 qf[QN];
#pragma unroll
    for (int s = 0; s < QN; ++s) qf[s] = *reinterpret_cast<const u32x4*>(qp + (2 * s + half) * (16 / (int)sizeof(T)));
    __builtin_amdgcn_sched_barrier(0);  // (asked for before the first keys, so that they need not be waited for together)

    f32x16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    float mx = -INFINITY, l = 0.f;
    bool far = false;
    float off = -kLift<TYPE>, times = a.scale2, limit = -INFINITY;  // p = 2^(score times - off); the maximum moves beyond the limit

    const unsigned k_lds = (unsigned)(unsigned long)(__attribute__((address_space(3))) char*)lds + wave * (2 * HALF), v_lds = k_lds + HALF;
    u32x4* lk = reinterpret_cast<u32x4*>(lds + wave * (2 * HALF));
    u32x4* lv = lk + kFewRows * PIECES;
    const int fr = lane / PIECES, fc = lane % PIECES;
    const unsigned kb = (unsigned)a.kts * (unsigned)sizeof(T), vb = (unsigned)a.vts * (unsigned)sizeof(T);
    // (rows behind the sequence repeat its last one: they are masked)
    auto fetch = [&](int j0, const T* from, unsigned pitch, unsigned to, bool keys) {
        const unsigned long long at = reinterpret_cast<unsigned long long>(from) + (unsigned long long)j0 * pitch;
        const int left = nk - 1 - j0;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int r = i * RW + fr;
            const unsigned piece = keys ? fc ^ k_flip<PIECES>(r) : sizeof(T) == 4 ? fc : fc ^ v_flip<PIECES>(r);
            lds_dma16(to + i * 1024, (unsigned)min(r, left) * pitch + piece * 16, at);
        }
    };
    if (begin < end) {
        fetch(t_first + 32 * begin, kp, kb, k_lds, true);
        fetch(t_first + 32 * begin, vp, vb, v_lds, false);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < QN; ++s) qf[s] = qf[s] ^ a.q_sign;
    for (int n = begin; n < end; ++n) {
        const int j0 = t_first + 32 * n;
        const bool masked = j0 < all_first || j0 + 32 > all_last, more = n + 1 < end;
        wait_vmcnt_imm<LOADS>();  // (the keys; the values asked for after them are still on their way)
        f32x16 sc;
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = 0.f;
#pragma unroll
        for (int s = 0; s < QN; ++s) {
            const u32x4 kf = lk[l31 * PIECES + ((2 * s + half) ^ k_flip<PIECES>(l31))];
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(kf[e]), __uint_as_float(qf[s][e]), sc, 0, 0, 0);
            } else
                sc = E::mfma(__builtin_bit_cast(typename E::V8, kf), __builtin_bit_cast(typename E::V8, qf[s]), sc);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the keys have been read)
        if (more) fetch(j0 + 32, kp, kb, k_lds, true);
        if (masked) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int j = j0 + 4 * half + 8 * (e >> 2) + (e & 3);
                sc[e] = j >= first && j < last ? sc[e] : -INFINITY;
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, sc[e]);
        top = fmaxf(top, __shfl_xor(top, 32)) * a.scale2;
        if (__any(top > limit)) {  // (as above)
            const float now = fmaxf(mx, top), f = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx - now);
            mx = now;
            far = __any(fabsf(now) > kFarTop && now != -INFINITY);
            off = (far || now == -INFINITY ? 0.f : now) - kLift<TYPE>, times = far ? 1.f : a.scale2, limit = far ? -INFINITY : now + 8.f;
            l *= f;
#pragma unroll
            for (int i = 0; i < DT; ++i) o[i] = o[i] * f;
            if (far) {
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[e] = scaled_below(sc[e], a.scale2, mx == -INFINITY ? 0.f : mx);
            }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            sc[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], times, -off));
            l += sc[e];
        }
        if (more)
            wait_vmcnt_imm<LOADS>();
        else
            wait_vmcnt_imm<0>();
        unsigned odd = 0;  // rows of V with infinities or NaN, in a masked step
        if (masked) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const bool bad = odd_value<TYPE>(lv[i * 64 + lane]);
                unsigned long long at = __ballot(bad);
                while (at) {  // (rare)
                    odd |= 1u << (i * RW + (__ffsll(at) - 1) / PIECES);
                    at &= at - 1;
                }
            }
            if (odd) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i)
                    if (odd >> (i * RW + fr) & 1) lv[i * 64 + lane] = u32x4{0, 0, 0, 0};
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
        }
        if constexpr (sizeof(T) == 4) {
            const float* vv = reinterpret_cast<const float*>(lv);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int j = 8 * (e >> 2) + 4 * half + (e & 3);
#pragma unroll
                for (int i = 0; i < DT; ++i) o[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(vv[j * D + 32 * i + l31], sc[e], o[i], 0, 0, 0);
            }
        } else {
            const char* vv = reinterpret_cast<const char*>(lv);
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                typename E::V8 pf;
#pragma unroll
                for (int e = 0; e < 8; ++e) pf[e] = (T)sc[8 * s + e];
#pragma unroll
                for (int i = 0; i < DT; ++i) {
                    union {
                        typename E::V8 v;
                        s16x4 p[2];
                    } vf;
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const int r = 16 * s + 8 * w + 4 * half + ((lane & 15) >> 2);
                        const int byte = 64 * i + (lane & 16) * 2 + (lane & 3) * 8;
                        vf.p[w] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) s16x4*)(vv + 16 * (r * PIECES + ((byte >> 4) ^ v_flip<PIECES>(r))) + (byte & 15)));
                    }
                    o[i] = E::mfma(vf.v, pf, o[i]);
                }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the values have been read)
        if (more) fetch(j0 + 32, vp, vb, v_lds, false);
        while (odd) {  // (uniform) only for the queries that see them
            const int j = __ffs(odd) - 1, at = j0 + j, e_at = (j >> 3) * 4 + (j & 3);
            odd &= odd - 1;
            float p = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (e == e_at) p = sc[e];
            p = __shfl(p, (j >> 2 & 1) * 32 + l31);
            if (at >= first && at < last) {
#pragma unroll
                for (int i = 0; i < DT; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        o[i][e] = fmaf(p, (float)vp[(long long)at * a.vts + 32 * i + 8 * (e >> 2) + 4 * half + (e & 3)], o[i][e]);
            }
        }
    }

    // the four waves' shares -> one
    l += __shfl_xor(l, 32);
    constexpr int PITCH = D + 4;
    float* so = reinterpret_cast<float*>(lds);
    float* sm = so + 4 * kFewRows * PITCH;  // [4][32], then the sums
    lds_barrier();                          // (keys and values are no longer read)
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<f32x4*>(so + (wave * kFewRows + l31) * PITCH + 32 * i + 2 * e + 4 * half) = f32x4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
    if (half == 0) {
        sm[wave * 32 + l31] = mx;
        sm[128 + wave * 32 + l31] = l;
    }
    lds_barrier();
    constexpr int W = D / 8;
    const int r = tid >> 3, c = (tid & 7) * 4;  // channels c + 32 i ..: eight neighbours read and write 128 bytes
    float all = -INFINITY, sum = 0.f, acc[W] = {};
#pragma unroll
    for (int w = 0; w < 4; ++w) all = fmaxf(all, sm[w * 32 + r]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float m = sm[w * 32 + r], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - all);
        sum += sm[128 + w * 32 + r] * f;  // (0 without a key; all scores NaN: NaN)
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(so + (w * kFewRows + r) * PITCH + 32 * i + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[4 * i + e] += x[e] * f;
        }
    }
    if (row0 + r >= rows) return;
    if (used <= 1) {
        const int tr = a.by_group(row0 + r), gr = row0 + r - tr * a.group;
        seen(a, tr + nk - nq, nk, first, last);
        const float inv = inverse_sum(sum, first < last);
        T* out = (T*)a.out + (long long)(q0 + tr) * a.ots + (long long)(h * a.group + gr) * a.ohs + c;
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            typedef T T4 __attribute__((ext_vector_type(4)));
            T4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (T)(acc[4 * i + e] * inv);
            *reinterpret_cast<T4*>(out + 32 * i) = y;
        }
    } else {
        const size_t at = (((size_t)tile * a.kv_heads + h) * a.splits + split) * kFewRows + r;
        if (c == 0) a.part_ml[at] = f32x2{all, sum};
#pragma unroll
        for (int i = 0; i < DT; ++i) *reinterpret_cast<f32x4*>(a.part_o + at * D + 32 * i + c) = f32x4{acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]};
    }
}

// The rows whose keys were split.  One workgroup per row: 16 groups of 16 lanes share its pieces.
template <int TYPE, int D>
__global__ __launch_bounds__(256) void attend_join_kernel(PackedArgs a) {
    using T = typename Elem<TYPE>::T;
    constexpr int W = D / 16;
    typedef float fw __attribute__((ext_vector_type(W)));
    __shared__ float part[16][D];
    const int x = blockIdx.x, r = x % kFewRows, back = a.by_kv_heads(x / kFewRows), h = x / kFewRows - back * a.kv_heads, tile = back;
    Place place;
    if (!find_tile<kFewRows>(a, tile, place) || place.row0 + r >= place.rows) return;
    int t_first, t_last, dummy, steps;
    few_seen(a, place, t_first, t_last, dummy, dummy);
    steps = (max(t_last - t_first, 0) + 31) / 32;
    const int used = few_used(steps, few_share(a, steps));
    if (used <= 1) return;  // (written already)
    const size_t at = ((size_t)tile * a.kv_heads + h) * a.splits * kFewRows + r;
    const int lane = threadIdx.x & 63, group = threadIdx.x >> 4, d = (threadIdx.x & 15) * W;
    // (at most 64 pieces: a lane for each)
    f32x2 ml = {-INFINITY, 0.f};
    if (lane < used) ml = a.part_ml[at + (size_t)lane * kFewRows];
    float all = ml[0];
#pragma unroll
    for (int o = 1; o < 64; o *= 2) all = fmaxf(all, __shfl_xor(all, o));
    const float f = ml[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[0] - all);
    float sum = ml[1] * f;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) sum += __shfl_xor(sum, o);
    const int tr = a.by_group(place.row0 + r), gr = place.row0 + r - tr * a.group;
    int first, last;
    seen(a, tr + place.nk - place.nq, place.nk, first, last);
    const float inv = inverse_sum(sum, first < last);
    fw acc;
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int s = 16 * i + group;
        const float fs = __shfl(f, s) * inv;
        if (s < used) {
            const fw y = *reinterpret_cast<const fw*>(a.part_o + (at + (size_t)s * kFewRows) * D + d);
#pragma unroll
            for (int e = 0; e < W; ++e) acc[e] = fmaf(y[e], fs, acc[e]);
        }
    }
    *reinterpret_cast<fw*>(&part[group][d]) = acc;
    __syncthreads();
    if (threadIdx.x < D) {
        float y = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) y += part[i][threadIdx.x];
        ((T*)a.out)[(long long)(place.q0 + tr) * a.ots + (long long)(h * a.group + gr) * a.ohs + threadIdx.x] = (T)y;
    }
}

struct PackedPlan {
    bool few;
    int tiles, splits;
    long long ml_bytes, bytes;
};
PackedPlan packed_plan(int type, long long q_rows, long long k_rows, int n_seqs, int heads, int kv_heads, int head_dim, int window) {
    const int group = heads / kv_heads;
    PackedPlan p;
    const long long wide = (q_rows * group / BM + n_seqs + 1) * kv_heads;  // workgroups of 128 rows (some without any)
    long long keys = n_seqs > 0 ? k_rows / n_seqs : 0;
    if (window > 0 && window < keys) keys = window;
    // 32 rows to a workgroup while that many of 128 are too few for 256 CUs.  fp32, where a tile takes longest: 3 x 256 tokens of
    // 8 heads of 64, window 8 (80 workgroups) 8.9 us against 20.9, 6000 of 8 / 2 heads of 128 (378) 706 / 778, 8192 (516) 1285 /
    // 1129.  16 bits, long sequences: 2048 tokens of 8 heads of 64 (144) 17.5 / 34.3, of 8 / 2 heads of 128 6000 (378) 132 / 132 and
    // 7000 (440) 171 / 159; short ones, where the beginning of a workgroup counts: 8 x 200 of 8 heads of 128 (168) 10.0 / 12.0,
    // 12 x 200 (248) 15.7 / 12.5.  And wherever a sequence's rows fill no more than one of 32: bf16, one token of 256 sequences of
    // 1 .. 2048, 32 / 8 heads of 128, 204 / 222, of 400 of 1 .. 300, 8 heads of 64, 25.6 / 39.5, 16 tokens of 128 of 1 .. 1000,
    // 8 heads of 128, 48.6 / 61.9; fp32, 128 of 1 .. 2048, 242 / 760.
    p.few = q_rows * group <= 32ll * n_seqs || wide <= (type == AFTER_T_F32 ? 512 : keys >= 1024 ? 384 : 192);
    p.tiles = (int)(q_rows * group / (p.few ? kFewRows : BM)) + n_seqs + 1;
    p.splits = 1;
    if (p.few) {
        // The keys are split where a quarter of the chip is not filled, at 512 keys and more to a workgroup.  bf16, 32 / 8 heads of
        // 128, one query: over 32768 keys 28.4 us against 276, over 2048 12.4 / 21.8, over 1024 12.5 / 13.1; 4 x one query over
        // 2000 16.5 / 22.5, 16 x (152 workgroups) 34.1 / 25.6.
        const long long fill = 512 / ((long long)p.tiles * kv_heads), most = keys / 512;
        if (fill >= 4) p.splits = (int)std::max(1ll, std::min(std::min(fill, most), 64ll));
    }
    const long long parts = p.splits > 1 ? (long long)p.tiles * kv_heads * p.splits * kFewRows : 0;
    p.ml_bytes = parts * 8;
    p.bytes = p.ml_bytes + parts * head_dim * 4;
    return p;
}

template <int TYPE, int D>
int run_packed(const PackedArgs& a, bool few, hipStream_t s) {
    using T = typename Elem<TYPE>::T;
    if (few) {
        constexpr size_t tiles = 8 * kFewRows * D * sizeof(T), joined = 4 * kFewRows * (D + 4) * 4 + 1024, lds = tiles > joined ? tiles : joined;
        static LdsAttr attr;
        AFTER_TRY(ensure_lds_attr(attr, (const void*)attend_few_kernel<TYPE, D>, lds));
        hipLaunchKernelGGL((attend_few_kernel<TYPE, D>), dim3((unsigned)a.tiles * a.kv_heads * a.splits), dim3(256), lds, s, a);
        if (a.splits > 1) hipLaunchKernelGGL((attend_join_kernel<TYPE, D>), dim3((unsigned)a.tiles * a.kv_heads * kFewRows), dim3(256), 0, s, a);
        AFTER_HIP_CHECK(hipGetLastError());
        return AFTER_OK;
    }
    constexpr size_t tiles = 4 * BN * D * sizeof(typename Elem<TYPE>::T), out = 4 * 32 * (D * sizeof(typename Elem<TYPE>::T) + 16), lds = tiles > out ? tiles : out;
    static LdsAttr attr;
    AFTER_TRY(ensure_lds_attr(attr, (const void*)attend_packed_kernel<TYPE, D>, lds));
    hipLaunchKernelGGL((attend_packed_kernel<TYPE, D>), dim3((unsigned)a.tiles * a.kv_heads), dim3(256), lds, s, a);
    AFTER_HIP_CHECK(hipGetLastError());
    return AFTER_OK;
}

}  // namespace
}  // namespace after

using namespace after;

static int check_sizes(int type, long long q_rows, long long k_rows, int n_seqs, int heads, int kv_heads, int head_dim, int window) {
    AFTER_REQUIRE(type == AFTER_T_F32 || type == AFTER_T_BF16 || type == AFTER_T_F16, AFTER_E_INVALID, "attend_packed: unknown element type %d", type);
    AFTER_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, AFTER_E_INVALID, "attend_packed: heads must be a multiple of kv_heads (got %d, %d)", heads,
                  kv_heads);
    AFTER_REQUIRE(head_dim == 64 || head_dim == 128, AFTER_E_INVALID, "attend_packed: head_dim 64 or 128 (got %d)", head_dim);
    AFTER_REQUIRE(n_seqs >= 0 && n_seqs <= (1 << 24) && q_rows >= 0 && q_rows < (1ll << 30) && k_rows >= 0 && k_rows < (1ll << 30), AFTER_E_INVALID,
                  "attend_packed: 0 <= n_seqs <= 2^24, 0 <= rows < 2^30");
    AFTER_REQUIRE(q_rows * (heads / kv_heads) < (1ll << 30), AFTER_E_INVALID, "attend_packed: q_rows x heads / kv_heads must stay below 2^30");
    const PackedPlan p = packed_plan(type, q_rows, k_rows, n_seqs, heads, kv_heads, head_dim, window);
    // (a grid's threads are counted in 32 bits)
    AFTER_REQUIRE(p.tiles < (1 << 24) / kv_heads, AFTER_E_INVALID, "attend_packed: too many tokens x heads for one call");
    return AFTER_OK;
}

extern "C" int after_attend_packed_workspace(int type, long long q_rows, long long k_rows, int n_seqs, int heads, int kv_heads, int head_dim, int window, long long* bytes) {
    AFTER_REQUIRE(bytes, AFTER_E_INVALID, "attend_packed_workspace: bytes is NULL");
    AFTER_TRY(check_sizes(type, q_rows, k_rows, n_seqs, heads, kv_heads, head_dim, window));
    *bytes = packed_plan(type, q_rows, k_rows, n_seqs, heads, kv_heads, head_dim, window).bytes;
    return AFTER_OK;
}

extern "C" int after_attend_packed(const after_packed* call, void* stream) {
    AFTER_REQUIRE(call, AFTER_E_INVALID, "attend_packed: no call");
    const after_packed& c = *call;
    AFTER_TRY(check_sizes(c.type, c.q_rows, c.k_rows, c.n_seqs, c.heads, c.kv_heads, c.head_dim, c.window));
    const int group = c.heads / c.kv_heads;
    AFTER_REQUIRE(std::isfinite(scale_log2(c.scale)) && !std::isnan(c.scale), AFTER_E_INVALID, "attend_packed: scale must be finite, times log2 e too");
    AFTER_REQUIRE(c.window >= 0 && c.chunk >= 1 && c.chunk <= (1 << 24) && (c.causal || (c.window == 0 && c.chunk == 1)), AFTER_E_INVALID,
                  "attend_packed: window >= 0 (0: none) and chunk >= 1, both for causal attention only");
    if (c.q_rows == 0) return AFTER_OK;
    const int per16 = 16 / (c.type == AFTER_T_F32 ? 4 : 2);
    const long long strides = c.q_token_stride | c.q_head_stride | c.k_token_stride | c.k_head_stride | c.v_token_stride | c.v_head_stride | c.out_token_stride | c.out_head_stride;
    AFTER_REQUIRE(c.q && c.out && c.q_starts && c.k_starts && (c.k_rows == 0 || (c.k && c.v)), AFTER_E_INVALID, "attend_packed: a pointer is NULL");
    AFTER_REQUIRE((((size_t)c.q | (size_t)c.k | (size_t)c.v | (size_t)c.out) & 15) == 0 && (strides & (per16 - 1)) == 0, AFTER_E_INVALID,
                  "attend_packed: q, k, v, out and their token and head strides must be multiples of 16 bytes");
    AFTER_REQUIRE(c.k_token_stride >= 0 && c.v_token_stride >= 0 && c.k_token_stride < (1 << 22) && c.v_token_stride < (1 << 22), AFTER_E_INVALID,
                  "attend_packed: the token strides of k and v must be below 2^22 elements");
    PackedArgs a;
    a.q = c.q, a.k = c.k, a.v = c.v, a.out = c.out, a.qs = c.q_starts, a.ks = c.k_starts;
    a.qts = c.q_token_stride, a.qhs = c.q_head_stride, a.kts = c.k_token_stride, a.khs = c.k_head_stride;
    a.vts = c.v_token_stride, a.vhs = c.v_head_stride, a.ots = c.out_token_stride, a.ohs = c.out_head_stride;
    a.q_rows = (int)c.q_rows, a.k_rows = (int)c.k_rows, a.n_seqs = c.n_seqs, a.kv_heads = c.kv_heads, a.group = group;
    PackedPlan p = packed_plan(c.type, c.q_rows, c.k_rows, c.n_seqs, c.heads, c.kv_heads, c.head_dim, c.window);
    AFTER_REQUIRE(!c.workspace || (((size_t)c.workspace & 15) == 0 && c.workspace_bytes >= p.bytes), AFTER_E_CAPACITY,
                  "attend_packed: a workspace has to be 16-byte aligned, here of %lld bytes (got %lld)", p.bytes, c.workspace_bytes);
    if (!c.workspace) p.splits = 1;
    a.tiles = p.tiles, a.splits = p.splits, a.by_splits = divisor(p.splits);
    a.part_ml = (f32x2*)c.workspace, a.part_o = (float*)((char*)c.workspace + p.ml_bytes);
    a.scale2 = scale_log2(c.scale);
    a.q_sign = c.scale < 0 ? (c.type == AFTER_T_F32 ? 0x80000000u : 0x80008000u) : 0u;
    a.causal = c.causal != 0, a.window = c.window < (1 << 30) ? c.window : 1 << 30, a.zero_rest = c.zero_rest;
    a.by_group = divisor(group), a.by_chunk = divisor(c.chunk), a.by_kv_heads = divisor(c.kv_heads);
    hipStream_t s = (hipStream_t)stream;
    if (c.head_dim == 64) {
        if (c.type == AFTER_T_F32) return run_packed<AFTER_T_F32, 64>(a, p.few, s);
        if (c.type == AFTER_T_BF16) return run_packed<AFTER_T_BF16, 64>(a, p.few, s);
        return run_packed<AFTER_T_F16, 64>(a, p.few, s);
    }
    if (c.type == AFTER_T_F32) return run_packed<AFTER_T_F32, 128>(a, p.few, s);
    if (c.type == AFTER_T_BF16) return run_packed<AFTER_T_BF16, 128>(a, p.few, s);
    return run_packed<AFTER_T_F16, 128>(a, p.few, s);
}
