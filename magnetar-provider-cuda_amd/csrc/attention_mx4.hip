// Attention over 4-bit stores (mx4.hpp), with the attention each key received
// on request.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(s_ij - m_i) / l_i,  s_ij = scale q_i . k_j
//
// over the keys j that query i admits, m_i and l_i the running maximum and sum
// of one pass over the keys. The matrix cores take the held keys and values as
// they are, one bf16 plane each, exactly; an f32 query or weight is split
// exactly into three bf16 planes (24 bits by truncation, 8 a plane), so a
// product is three matrix instructions with f32 sums. Scores, statistics and
// outputs stay in f32.
//
// Query heads that share a KV head are rows of one product: row r of a KV head
// is head r % group of query r / group. What follows holds for few rows, where
// reading the stores bounds the call; prompts, bound by their products, have a
// kernel of their own below, with the scores from block-scaled products. A wave
// takes 16 rows and 64 keys at a time (16x16x32 products), and both products are
// fed from the stores' units as they lie in memory. With kg a group of four keys, n a lane of 16 and g one
// of the wave's four lane groups:
//
//   scores   A = K: lane (m, g) holds keys 4 m + i for product i (the four rows
//            of group kg = m), and of each key the units n = 4 t + g, t < 4; the
//            columns of a step go by the order of the unit's bytes, in which Q
//            is laid out once.
//            C: lane (q, g), register r: key 16 g + 4 r + i of row q.
//   outputs  A = V^T: lane (n, g) holds column 16 c + n of the groups kg = 4 g +
//            r: keys 16 g + 4 r + i. B = P^T is then lane (q, g)'s own scores.
//            C: lane (q, g), register r: column 16 c + 4 g + r of row q.
//
// so neither the weights nor the values pass through LDS, and a row's maximum
// and its rescaling are its own lane's.
//
// Up to four rows (a token of up to four query heads a KV head) leave twelve of
// the sixteen columns empty: there the planes take columns of their own, column
// 4 * plane + row (the fourth plane is zero), and a product is one matrix
// instruction instead of three. Scores are added up over the planes' lanes, the
// outputs once at the end.
#include <cmath>

#include "mx4.hpp"

namespace {

using mhip::bf16x2;
using mhip::bf16x8;
using mhip::f32x2;
using mhip::f32x4;
using mhip::Mx4Unit;

constexpr float kLog2e = 1.4426950408889634f;

struct Mx4Attn {
    const float* q;
    const uint8_t *k, *v;
    float* out;
    uint64_t q_bs, o_bs;          // floats between sequences
    uint64_t k_bs, v_bs;          // bytes between sequences' stores
    uint64_t code_bytes;          // of one store
    uint64_t q_ld;                // floats between queries: heads * d
    const uint64_t* advance;      // captured step: replay offset added to the key count
    int seq, kv, rows;            // queries, keys, rows of a KV head (seq * group)
    int heads, kv_heads, group, d, groups;
    int causal, window;           // window -1: none
    int vec;                      // rows of q and out are whole float4s
    int vec_q;                    // rows of q are whole float4s
    int row_tiles, heavy_ranks, chunks, chunk_tiles, batch;
    float c;                      // scale * log2(e)
    char* planes;                 // [batch][kv head][32 rows] SumCfg::kBytes (weights asked for)
    uint64_t planes_ld;
    float* part_o;                // [batch][kv head][row tile][chunk][row][DP]
    float* part_ml;               // [batch][kv head][row tile][chunk][row][2]
    uint32_t* arrived;            // [batch][kv head][row tile]: chunks done, 0 between calls
    float* stats;                 // [batch][kv head][rows][2]: m and 1 / l (weights asked for)
    float* kept;                  // [batch][kv head][rows][kept_ld]: scores (weights asked for, one row tile)
    uint64_t kept_ld;
};

// The keys [lo, hi) that a row's query admits, and those that all rows of a
// tile do.
struct Keys {
    int lo, hi;
};
__device__ __forceinline__ bool outside(const Keys& k, int key) {  // one comparison
    return static_cast<uint32_t>(key - k.lo) >= static_cast<uint32_t>(k.hi - k.lo);
}
__device__ __forceinline__ Keys row_keys(const Mx4Attn& a, int kv, int row) {
    const int at = kv - a.seq + row / a.group;
    Keys k;
    k.hi = a.causal ? at + 1 : kv;
    k.lo = a.window > 0 ? max(at - (a.window - 1), 0) : 0;
    return k;
}

__device__ __forceinline__ uint32_t top16(float hi, float lo) {  // their upper halves: {lo, hi}
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ float truncated(float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFF0000u); }

union Frag {
    uint32_t u[4];
    bf16x8 v;
};

// x[0..8) into three bf16 planes that add up to it exactly: what a truncation
// to 8 bits leaves has 16 bits, and what that leaves has 8.
__device__ __forceinline__ void split8(const float (&x)[8], Frag (&f)[3]) {
#pragma unroll
    for (int y = 0; y < 4; ++y) {
        const float a = x[2 * y], b = x[2 * y + 1];
        const float a1 = a - truncated(a), b1 = b - truncated(b);
        const float a2 = a1 - truncated(a1), b2 = b1 - truncated(b1);
        f[0].u[y] = top16(b, a);
        f[1].u[y] = top16(b1, a1);
        f[2].u[y] = top16(b2, a2);
    }
}

__device__ __forceinline__ f32x4 mfma(const Frag& a, const Frag& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t bits(bf16x2 v) {
    uint32_t u;
    __builtin_memcpy(&u, &v, 4);
    return u;
}

// The plane that a lane of the few-rows form has: x less the part that the
// planes before it hold. The masks of plane 3 leave x - x, zero.
struct Plane {
    uint32_t m1, m2;
};
__device__ __forceinline__ Plane plane_of(int slot) {
    return Plane{slot == 0 ? 0u : slot == 3 ? 0xFFFFFFFFu : 0xFFFF0000u, slot == 2 ? 0xFFFF0000u : 0u};
}
__device__ __forceinline__ float plane_part(float x, Plane p) {
    x -= __uint_as_float(__float_as_uint(x) & p.m1);
    return x - __uint_as_float(__float_as_uint(x) & p.m2);
}
__device__ __forceinline__ void plane8(const float (&x)[8], Plane p, Frag& f) {
#pragma unroll
    for (int y = 0; y < 4; ++y) f.u[y] = top16(plane_part(x[2 * y + 1], p), plane_part(x[2 * y], p));
}

// x summed over the lanes n, n + 4, n + 8 and n + 12 of 16.
__device__ __forceinline__ float sum_planes(float x) {
    x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x128, 0xF, 0xF, true));  // row_ror:8
    return x + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x124, 0xF, 0xF, true));  // row_ror:4
}

// The operand of a product's rows: FEW one plane a lane, else all three.
template <bool FEW>
struct Rows {
    Frag f[FEW ? 1 : 3];
};
template <bool FEW>
__device__ __forceinline__ void rows8(const float (&x)[8], Plane p, Rows<FEW>& w) {
    if constexpr (FEW)
        plane8(x, p, w.f[0]);
    else
        split8(x, w.f);
}
template <bool FEW>
__device__ __forceinline__ f32x4 product(const Frag& a, const Rows<FEW>& w, f32x4 c) {
    if constexpr (!FEW) {
        c = mfma(a, w.f[2], c);
        c = mfma(a, w.f[1], c);
    }
    return mfma(a, w.f[0], c);
}

// Row `row`'s part of Q for lane group g: step s, pair y takes byte x = 4 s + y
// of the lane group's units in order (unit n = 4 t + g of t = x / NB, block p =
// x % NB): columns 32 p + n and 32 p + 16 + n.
template <int NB, bool FEW>
__device__ __forceinline__ void load_q(const Mx4Attn& a, const float* qrow, int g, Plane plane, Rows<FEW> (&q)[NB]) {
#pragma unroll
    for (int s = 0; s < NB; ++s) {
        float x[8];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const int t = (4 * s + y) / NB, p = (4 * s + y) % NB;
            const int col = 32 * p + 4 * t + g;
            const float x0 = qrow[min(col, a.d - 1)], x1 = qrow[min(col + 16, a.d - 1)];
            x[2 * y] = col < a.d ? x0 : 0.0f;
            x[2 * y + 1] = col + 16 < a.d ? x1 : 0.0f;
        }
        rows8<FEW>(x, plane, q[s]);
    }
}

// The stores' units of 64 keys for one lane. Groups past the last are read as
// the last one: their keys are masked.
template <int NB>
struct Strip {
    Mx4Unit<NB> unit[4], scale[4];
};
template <int NB>
__device__ __forceinline__ void load_k(const uint32_t* codes, const uint32_t* scales, int kg0, int last, int m, int g,
                                       Strip<NB>& k) {
    const int kg = min(kg0 + m, last);
#pragma unroll
    for (int t = 0; t < 4; ++t) k.unit[t] = mhip::mx4_load<NB>(codes + (static_cast<uint64_t>(kg) * 16 + 4 * t + g) * NB);
    k.scale[0] = mhip::mx4_load<NB>(scales + static_cast<uint64_t>(kg) * NB);
}
template <int NB>
__device__ __forceinline__ void load_v(const uint32_t* codes, const uint32_t* scales, int kg0, int last, int n, int g,
                                       Strip<NB>& v) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int kg = min(kg0 + 4 * g + r, last);
        v.unit[r] = mhip::mx4_load<NB>(codes + (static_cast<uint64_t>(kg) * 16 + n) * NB);
        v.scale[r] = mhip::mx4_load<NB>(scales + static_cast<uint64_t>(kg) * NB);
    }
}

// S^T of 64 keys: st[i][r] is key 16 g + 4 r + i of the lane's row.
template <int NB, bool FEW>
__device__ __forceinline__ void scores(const Strip<NB>& k, const Rows<FEW> (&q)[NB], f32x4 (&st)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < NB; ++s) {
            Frag f;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int t = (4 * s + y) / NB, p = (4 * s + y) % NB, at = i * NB + p;
                f.u[y] = bits(mhip::mx4_bf16(k.unit[t].w[at / 4], mhip::mx4_scale(k.scale[0].w[p], i), at % 4));
            }
            acc = product<FEW>(f, q[s], acc);
        }
        if constexpr (FEW)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = sum_planes(acc[r]);
        st[i] = acc;
    }
}

// O^T += V^T P^T over 64 keys, p as scores() left them.
template <int NB, bool FEW>
__device__ __forceinline__ void outputs(const Strip<NB>& v, const float (&p)[4][4], Plane plane, f32x4 (&o)[2 * NB]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {  // 32 keys: r = 2 u and 2 u + 1
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = p[j % 4][2 * u + j / 4];
        Rows<FEW> w;
        rows8<FEW>(x, plane, w);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            Frag lo, hi;  // columns 32 b + n and 32 b + 16 + n
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int r = 2 * u + y / 2, i = 2 * (y % 2), at0 = i * NB + b, at1 = at0 + NB;
                const uint32_t k0 = bits(mhip::mx4_bf16(v.unit[r].w[at0 / 4], mhip::mx4_scale(v.scale[r].w[b], i), at0 % 4));
                const uint32_t k1 = bits(mhip::mx4_bf16(v.unit[r].w[at1 / 4], mhip::mx4_scale(v.scale[r].w[b], i + 1), at1 % 4));
                lo.u[y] = __builtin_amdgcn_perm(k1, k0, 0x05040100u);
                hi.u[y] = __builtin_amdgcn_perm(k1, k0, 0x07060302u);
            }
            o[2 * b] = product<FEW>(lo, w, o[2 * b]);
            o[2 * b + 1] = product<FEW>(hi, w, o[2 * b + 1]);
        }
    }
}

__device__ __forceinline__ uint32_t bytes_255(uint32_t x) {  // bit 7 of each byte that is 255
    return ((x & 0x7F7F7F7Fu) + 0x01010101u) & x & 0x80808080u;
}
// ... a bit each, byte i's bit i.
__device__ __forceinline__ uint32_t byte_bits(uint32_t ff) {
    return (ff >> 7 & 1u) | (ff >> 14 & 2u) | (ff >> 21 & 4u) | (ff >> 28 & 8u);
}
__device__ __forceinline__ uint32_t whole_bytes(uint32_t ff) { return ff | (ff - (ff >> 7)); }

// In a strip at a mask's edge a value that is no number may belong to a key
// that some rows admit and others do not, and to the product 0 times it is no
// number for all of them. Its block is taken out of the strip (scale byte 0:
// finite) and, for the rows that admit the key, put into the sums of its
// columns. `base`: the strip's first key; keys from `hi` on belong to no row.
template <int NB>
__device__ __forceinline__ void edge_values(Strip<NB>& v, int base, int g, const Keys& row, int hi, f32x4 (&o)[2 * NB]) {
    uint32_t flags[NB];  // bit 4 r + i: the block of key 16 g + 4 r + i is no number
    uint32_t any = 0;
#pragma unroll
    for (int b = 0; b < NB; ++b) flags[b] = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int live = min(max(hi - (base + 16 * g + 4 * r), 0), 4);  // keys of the unit before `hi`
        const uint32_t keep = static_cast<uint32_t>((1ull << (8 * live)) - 1);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint32_t scale = v.scale[r].w[b] & keep, ff = bytes_255(scale);
            v.scale[r].w[b] = scale & ~whole_bytes(ff);
            flags[b] |= byte_bits(ff) << (4 * r);
            any |= ff;
        }
    }
    if (__ballot(any != 0) == 0) return;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        bool hit = false;
#pragma unroll
        for (int gg = 0; gg < 4; ++gg)
            for (uint32_t keys = __builtin_amdgcn_readlane(flags[b], 16 * gg); keys != 0; keys &= keys - 1) {
                const int key = base + 16 * gg + __builtin_ctz(keys);
                if (key >= row.lo && key < row.hi) hit = true;
            }
        if (hit) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[2 * b][e] = o[2 * b + 1][e] = NAN;
        }
    }
}

// Row `row`'s place in q or out.
__device__ __forceinline__ uint64_t row_at(const Mx4Attn& a, int kvh, int row) {
    const int i = row / a.group, head = kvh * a.group + row % a.group;
    return static_cast<uint64_t>(i) * a.q_ld + static_cast<uint64_t>(head) * a.d;
}

constexpr int kMaxChunks = 256;
// Waves of a rows workgroup: eight, of a head of more than four blocks four
// (their sums in LDS are 16 rows a wave).
template <bool FEW>
constexpr int kRowTile = FEW ? 4 : 16;
template <int NB>
constexpr int kRowWaves = NB > 4 ? 4 : 8;

// One row's outputs for four columns.
__device__ __forceinline__ void store_out(const Mx4Attn& a, int b, int kvh, int row, int col, f32x4 o) {
    float* dst = a.out + b * a.o_bs + row_at(a, kvh, row) + col;
    if (a.vec) {
        if (col < a.d) *reinterpret_cast<f32x4*>(dst) = o;
    } else {
#pragma unroll
        for (int x = 0; x < 4; ++x)
            if (col + x < a.d) dst[x] = o[x];
    }
}

// Chunk records pass between workgroups whose L2 caches differ. They go past
// the caches, as stores and loads at device scope, 8 bytes each: a store is
// done once vmcnt has counted it, and only then does its workgroup count itself
// in. (Plain stores under a device fence took 100-140 us more with 512-1024
// workgroups: every fence writes a whole L2 back.)
__device__ __forceinline__ void put2(float* p, float x, float y) {
    const uint64_t v = static_cast<uint64_t>(__float_as_uint(y)) << 32 | __float_as_uint(x);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x2 get2(const float* p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return f32x2{__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32))};
}

// A workgroup: 16 rows of a KV head (FEW: 4) over one chunk of their keys, the chunk's
// 64-key strips dealt to the waves in turn, the waves' sums added up in LDS.
// The chunks split the keys that the tile's rows admit evenly; how many there
// are goes by the store's capacity, how long they are by the key count, which a
// replay moves. Of several chunks the workgroup that ends last adds up the
// records of all, in their order, each weighted by 2 to its maximum less the
// largest: one launch, and the same bits whichever it is.
//
// The next strip's keys are loaded once the scores have taken this one's, its
// values once the outputs have: both loads run under the other product, in the
// registers that it has freed.
//
// Measured (heads of 128): 131073 keys of 8 KV heads, 143 MB, in 33 us, 4.3 TB/s;
// 8 sequences of 4096 keys, 36 MB, in 15 us: 3.7 for the first loads, 8 for two
// strips a wave, 1.4 for the records and the count, 2.4 for the merge. A single
// short one 6 us, its loads' and barriers' latency.
template <int NB, bool FEW>
__global__ __launch_bounds__(64 * kRowWaves<NB>) void mx4_rows_kernel(Mx4Attn a) {
    constexpr int DP = 32 * NB, kWaves = kRowWaves<NB>, kThreads = 64 * kWaves, RT = kRowTile<FEW>;
    union Lds {
        struct {
            float o[kWaves][RT][DP + 4];
        } waves;
        struct {
            float factor[RT][kMaxChunks];
            f32x4 sum[kThreads];
            float l[RT];
        } merge;
    };
    __shared__ Lds lds;
    __shared__ float lds_m[kWaves][RT], lds_l[kWaves][RT];
    __shared__ uint32_t lds_last;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int chunk = a.chunks > 1 ? blockIdx.x % a.chunks : 0, tile = a.chunks > 1 ? blockIdx.x / a.chunks : blockIdx.x;
    const int kvh = blockIdx.y, b = blockIdx.z;
    const int kv = a.kv + (a.advance ? static_cast<int>(*a.advance) : 0);

    const int row0 = tile * RT, row_last = min(row0 + RT - 1, a.rows - 1), live = row_last - row0 + 1;
    const int slot = n / RT, own = n % RT, row = min(row0 + own, row_last);
    const Plane plane = plane_of(slot);
    const Keys mine = row_keys(a, kv, row), head = row_keys(a, kv, row0), tail = row_keys(a, kv, row_last);
    const int begin = head.lo / 64, end = (tail.hi + 63) / 64;  // strips
    const int per = a.chunks > 1 ? (end - begin + a.chunks - 1) / a.chunks : end - begin;
    const int s0 = begin + chunk * per, s1 = min(s0 + per, end);

    const uint8_t* ks = a.k + b * a.k_bs;
    const uint8_t* vs = a.v + b * a.v_bs;
    const uint64_t head_units = static_cast<uint64_t>(kvh) * a.groups;
    const uint32_t* kc = reinterpret_cast<const uint32_t*>(ks) + head_units * 16 * NB;
    const uint32_t* kx = reinterpret_cast<const uint32_t*>(ks + a.code_bytes) + head_units * NB;
    const uint32_t* vc = reinterpret_cast<const uint32_t*>(vs) + head_units * 16 * NB;
    const uint32_t* vx = reinterpret_cast<const uint32_t*>(vs + a.code_bytes) + head_units * NB;
    const int last = (kv - 1) / 4;

    Strip<NB> k, v;
    int s = s0 + wave;
    load_k<NB>(kc, kx, s * 16, last, n, g, k);
    load_v<NB>(vc, vx, s * 16, last, n, g, v);
    Rows<FEW> q[NB];
    load_q<NB, FEW>(a, a.q + b * a.q_bs + row_at(a, kvh, row), g, plane, q);

    f32x4 o[2 * NB];
#pragma unroll
    for (int c = 0; c < 2 * NB; ++c) o[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    for (; s < s1; s += kWaves) {
        const int base = 64 * s;
        f32x4 st[4];
        scores<NB, FEW>(k, q, st);
        load_k<NB>(kc, kx, (s + kWaves) * 16, last, n, g, k);
        if (a.kept && n < live) {
            float* to = a.kept + ((static_cast<uint64_t>(b) * a.kv_heads + kvh) * a.rows + row) * a.kept_ld + base + 16 * g;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *reinterpret_cast<f32x4*>(to + 4 * r) = f32x4{st[0][r], st[1][r], st[2][r], st[3][r]};
        }
        if (base < tail.lo || base + 64 > head.hi) {
            asm volatile("");  // a branch
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = base + 16 * g + 4 * r + i;
                    if (outside(mine, key)) st[i][r] = -INFINITY;
                }
            edge_values<NB>(v, base, g, mine, tail.hi, o);
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, st[i][r]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float m_new = fmaxf(m, top * a.c);
        const float m_use = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m - m_use);
        m = m_new;
        float p[4][4], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[i][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i][r], a.c, -m_use));
                sum += p[i][r];
            }
        l = l * alpha + sum;
        if (__ballot(alpha != 1.0f) != 0) {
#pragma unroll
            for (int c = 0; c < 2 * NB; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[c][e] *= alpha;
        }
        outputs<NB, FEW>(v, p, plane, o);
        load_v<NB>(vc, vx, (s + kWaves) * 16, last, n, g, v);
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    if (g == 0 && slot == 0) lds_m[wave][own] = m;
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, lds_m[w][own]);
    const float f = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top));
#pragma unroll
    for (int c = 0; c < 2 * NB; ++c) {
        if constexpr (FEW)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[c][e] = sum_planes(o[c][e]);
        if (slot == 0) *reinterpret_cast<f32x4*>(&lds.waves.o[wave][own][16 * c + 4 * g]) = o[c] * f;
    }
    if (g == 0 && slot == 0) lds_l[wave][own] = l * f;
    __syncthreads();

    const uint64_t tile_id = (static_cast<uint64_t>(b) * a.kv_heads + kvh) * a.row_tiles + tile;
    const uint64_t rec = tile_id * a.chunks + chunk;
    if (a.chunks > 1) {
        // Two columns a lane: a wave's stores fill whole lines.
        for (int e = threadIdx.x; e < live * (DP / 2); e += kThreads) {
            const int r = e / (DP / 2), col = e % (DP / 2) * 2;
            f32x2 sum = {0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) sum += *reinterpret_cast<const f32x2*>(&lds.waves.o[w][r][col]);
            put2(a.part_o + (rec * RT + r) * DP + col, sum.x, sum.y);
        }
    } else {
        for (int e = threadIdx.x; e < live * (DP / 4); e += kThreads) {
            const int r = e / (DP / 4), col = e % (DP / 4) * 4;
            f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
            float total = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                sum += *reinterpret_cast<const f32x4*>(&lds.waves.o[w][r][col]);
                total += lds_l[w][r];
            }
            store_out(a, b, kvh, row0 + r, col, sum * (1.0f / total));
        }
    }
    if (threadIdx.x < live) {
        float total = 0.0f, mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            total += lds_l[w][threadIdx.x];
            mx = fmaxf(mx, lds_m[w][threadIdx.x]);
        }
        if (a.chunks > 1) {
            put2(a.part_ml + (rec * RT + threadIdx.x) * 2, mx, total);
        } else if (a.stats) {
            float* st = a.stats + ((static_cast<uint64_t>(b) * a.kv_heads + kvh) * a.rows + row0 + threadIdx.x) * 2;
            st[0] = mx == -INFINITY ? 0.0f : mx;
            st[1] = 1.0f / total;
        }
    }
    if (a.chunks == 1) return;

    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) lds_last = atomicInc(&a.arrived[tile_id], a.chunks - 1) == static_cast<uint32_t>(a.chunks) - 1;
    __syncthreads();
    if (!lds_last) return;

    // Four columns a thread; where those are few, `ways` threads share a cell's
    // chunks. The first records are on their way while the rows' maxima are found.
    constexpr int kAhead = 8;
    const int cells = live * (DP / 4);
    int ways = 1;
    while (ways * 2 * cells <= kThreads) ways *= 2;
    const float* records = a.part_o + tile_id * a.chunks * RT * DP;
    auto record = [&](int cell, int c) {
        const float* at = records + static_cast<uint64_t>(c) * RT * DP + cell * 4;
        const f32x2 x = get2(at), y = get2(at + 2);
        return f32x4{x.x, x.y, y.x, y.y};
    };
    const int cell0 = static_cast<int>(threadIdx.x) % cells, way = static_cast<int>(threadIdx.x) / cells;
    f32x4 ahead[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
        const int c = way + j * ways;
        ahead[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (way < ways && c < a.chunks) ahead[j] = record(cell0, c);
    }
    // kThreads / RT threads a row, at most a wave.
    {
        constexpr int kPer = kThreads / RT < 64 ? kThreads / RT : 64, kOwn = kMaxChunks / kPer;
        const int r = threadIdx.x / kPer, c0 = threadIdx.x % kPer;
        const float* ml = a.part_ml + (tile_id * a.chunks * RT + r) * 2;
        f32x2 rec_ml[kOwn];
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
            const int c = c0 + j * kPer;
            rec_ml[j] = f32x2{-INFINITY, 0.0f};
            if (r < live && c < a.chunks) rec_ml[j] = get2(ml + c * 2 * RT);
        }
#pragma unroll
        for (int j = 0; j < kOwn; ++j) mx = fmaxf(mx, rec_ml[j].x);
#pragma unroll
        for (int off = 1; off < kPer; off *= 2) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
        const float m_use = mx == -INFINITY ? 0.0f : mx;
        float total = 0.0f;
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
            const int c = c0 + j * kPer;
            const float fc = __builtin_amdgcn_exp2f(rec_ml[j].x - m_use);
            if (r < live && c < a.chunks) lds.merge.factor[r][c] = fc;
            total += rec_ml[j].y * fc;
        }
#pragma unroll
        for (int off = 1; off < kPer; off *= 2) total += __shfl_xor(total, off, 64);
        if (r < live && c0 == 0) {
            lds.merge.l[r] = 1.0f / total;
            if (a.stats) {
                float* st = a.stats + ((static_cast<uint64_t>(b) * a.kv_heads + kvh) * a.rows + row0 + r) * 2;
                st[0] = m_use;
                st[1] = 1.0f / total;
            }
        }
    }
    __syncthreads();
    for (int cell = cell0; cell < cells; cell += kThreads) {  // more than one only where ways is 1
        const int r = cell / (DP / 4), col = cell % (DP / 4) * 4;
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        int c = way;
        if (cell == cell0) {
#pragma unroll
            for (int j = 0; j < kAhead; ++j, c += ways)
                if (way < ways && c < a.chunks) sum += ahead[j] * lds.merge.factor[r][c];
        }
        if (way < ways)
#pragma unroll 4
            for (; c < a.chunks; c += ways) sum += record(cell, c) * lds.merge.factor[r][c];
        if (ways > 1) {
            lds.merge.sum[threadIdx.x] = sum;
            __syncthreads();
            if (way == 0)
                for (int w = 1; w < ways; ++w) sum += lds.merge.sum[w * cells + cell];
        }
        if (way == 0) store_out(a, b, kvh, row0 + r, col, sum * lds.merge.l[r]);
    }
}

// ---------------------------------------------------------------------------
// Prompts
// ---------------------------------------------------------------------------

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x32 __attribute__((ext_vector_type(32)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));

__device__ __forceinline__ f32x16 mfma32(const Frag& a, const Frag& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}

// The scores of a prompt come from the block-scaled matrix instructions, which
// take K's codes and scale bytes as they are held, and Q as planes of six bits
// (E2M3: with magnitudes below 2 under its scale, multiples of 1/8). A plane is
// the nearest to what the planes before it leave, at most 1/16 of their unit,
// so each adds five bits: six planes hold a block of 32 values of Q to within
// 2^-30 of its largest one, and add up in f32, the smallest first. Six such
// products take the time of one and a half in bf16, and K needs no conversion.
// (Five planes: 6.7e-8 of the scores' norm off, an f32 chain of multiply-adds
// 1.4e-7, six 3.0e-8; with one value of a block 1000 times the others and keys
// that are zero there, 2.6e-5 and 7.9e-7.)
constexpr int kQPlanes = 6;
template <int NB>
struct QPlanes {
    static constexpr int kSteps = (NB + 1) / 2;  // of two blocks, one a half of the wave
    // Above two blocks the registers do not hold all: planes 3 to 5 stay in LDS.
    static constexpr bool kLow = NB > 2;
    u32x6 f[kSteps][kQPlanes];
    uint32_t scale[kSteps][2];  // scale bytes of planes 0-3 and 4-5
};

// A plane of one lane in LDS, 16 and 8 bytes side by side over the lanes
// (`p`: the plane's place, at the lane's 16 bytes).
constexpr int kPlaneBytes = 64 * 24;
__device__ __forceinline__ void store_plane(char* p, const u32x6& f) {
    const uint4 x = {f[0], f[1], f[2], f[3]};
    const uint2 y = {f[4], f[5]};
    *reinterpret_cast<uint4*>(p) = x;
    *reinterpret_cast<uint2*>(p + 1024 - 8 * (threadIdx.x & 63)) = y;
}
__device__ __forceinline__ u32x6 load_plane(const char* p) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    const uint2 y = *reinterpret_cast<const uint2*>(p + 1024 - 8 * (threadIdx.x & 63));
    return u32x6{x.x, x.y, x.z, x.w, y.x, y.y};
}

// Lane (row, h), step s: block 2 s + h of the row (32 NB values in LDS, zeros
// past d), its values 2 i and 2 i + 1 the block's columns i and 16 + i, as the
// codes of K lie.
template <int NB>
__device__ __forceinline__ void make_q_planes(const float* qrow, int h, QPlanes<NB>& q) {
#pragma unroll
    for (int s = 0; s < QPlanes<NB>::kSteps; ++s) {
        const int p = 2 * s + h;
        f32x16 lo, hi;
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(qrow + 32 * min(p, NB - 1) + 4 * i);
            const f32x4 y = *reinterpret_cast<const f32x4*>(qrow + 32 * min(p, NB - 1) + 16 + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                lo[4 * i + e] = p < NB ? x[e] : 0.0f;
                hi[4 * i + e] = p < NB ? y[e] : 0.0f;
                top = max(top, max(__float_as_uint(lo[4 * i + e]) & 0x7FFFFFFFu, __float_as_uint(hi[4 * i + e]) & 0x7FFFFFFFu));
            }
        }
        // Magnitudes below 2 under 2^(e - 127), the last plane's byte above 0.
        const uint32_t e = max(top >> 23, 5u * kQPlanes);
        const bool nan = top >= 0x7F800000u;
        uint32_t bytes[2] = {0, 0};
#pragma unroll
        for (int n = 0; n < kQPlanes; ++n) {
            const uint32_t en = e - 5 * n;
            const float scale = __uint_as_float(en << 23);
            q.f[s][n] = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(lo, hi, scale);
            bytes[n / 4] |= (nan ? 255u : en) << (8 * (n % 4));
            if (n + 1 < kQPlanes) {
                const f32x32 held = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(q.f[s][n], scale);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    lo[i] -= held[2 * i];
                    hi[i] -= held[2 * i + 1];
                }
            }
        }
        q.scale[s][0] = bytes[0];
        q.scale[s][1] = bytes[1];
    }
}

// Four columns of a row of q, zeros past d.
__device__ __forceinline__ f32x4 load_q4(const Mx4Attn& a, const float* qrow, int col) {
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (a.vec_q) {
        if (col < a.d) x = *reinterpret_cast<const f32x4*>(qrow + col);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < a.d) x[e] = qrow[col + e];
    }
    return x;
}

// c += K (32 keys, block 2 s + h a lane half) by plane N of Q.
template <int OPK, int OPQ>
__device__ __forceinline__ f32x16 scaled_product(const Frag& k, uint32_t kscale, const u32x6& q, uint32_t qscale, f32x16 c) {
    const i32x8 x = {static_cast<int>(k.u[0]), static_cast<int>(k.u[1]), static_cast<int>(k.u[2]), static_cast<int>(k.u[3]), 0, 0, 0, 0};
    const i32x8 y = {static_cast<int>(q[0]), static_cast<int>(q[1]), static_cast<int>(q[2]),
                     static_cast<int>(q[3]), static_cast<int>(q[4]), static_cast<int>(q[5]), 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 2, OPK, static_cast<int>(kscale), OPQ, static_cast<int>(qscale));
}
// st[0] and st[1] (two chains) += 32 keys each by all planes of Q, the smallest
// first. `low`: planes 3 to 5 of the step, from LDS.
template <int OPK, int NB>
__device__ __forceinline__ void score_step(const Frag& k0, const Frag& k1, uint32_t s0, uint32_t s1, const QPlanes<NB>& q, int s,
                                           const char* low, f32x16 (&st)[2]) {
    u32x6 f[3];
#pragma unroll
    for (int n = 0; n < 3; ++n) {
        if constexpr (QPlanes<NB>::kLow)
            f[n] = load_plane(low + (3 * s + n) * kPlaneBytes);
        else
            f[n] = q.f[s][3 + n];
    }
    st[0] = scaled_product<OPK, 1>(k0, s0, f[2], q.scale[s][1], st[0]);
    st[1] = scaled_product<OPK, 1>(k1, s1, f[2], q.scale[s][1], st[1]);
    st[0] = scaled_product<OPK, 0>(k0, s0, f[1], q.scale[s][1], st[0]);
    st[1] = scaled_product<OPK, 0>(k1, s1, f[1], q.scale[s][1], st[1]);
    st[0] = scaled_product<OPK, 3>(k0, s0, f[0], q.scale[s][0], st[0]);
    st[1] = scaled_product<OPK, 3>(k1, s1, f[0], q.scale[s][0], st[1]);
    st[0] = scaled_product<OPK, 2>(k0, s0, q.f[s][2], q.scale[s][0], st[0]);
    st[1] = scaled_product<OPK, 2>(k1, s1, q.f[s][2], q.scale[s][0], st[1]);
    st[0] = scaled_product<OPK, 1>(k0, s0, q.f[s][1], q.scale[s][0], st[0]);
    st[1] = scaled_product<OPK, 1>(k1, s1, q.f[s][1], q.scale[s][0], st[1]);
    st[0] = scaled_product<OPK, 0>(k0, s0, q.f[s][0], q.scale[s][0], st[0]);
    st[1] = scaled_product<OPK, 0>(k1, s1, q.f[s][0], q.scale[s][0], st[1]);
}

constexpr uint64_t kMinChunk = 8;  // key tiles
constexpr float kLag = 8.0f;       // by which a score passes the maximum before it moves
constexpr int kPromptWaves = 4, kPromptRows = 32 * kPromptWaves;

// Four waves of 32 rows share tiles of 64 keys in LDS, each thread carrying one
// unit of K and one of V there from the stores:
//
//   K as codes, [half of 32 keys][block][key] 16 bytes (the blocks 16 bytes
//     apart in the banks). A unit has one byte of each of 4 NB (key, block)
//     pairs; four lanes transpose theirs to write four bytes of a pair at once.
//     Behind them a key's scale bytes, a dword for four blocks.
//   V as bf16 operands of 32x32x16 products, [half][step of 16 keys][block][lane]
//     16 bytes, lane (m, h) the keys 4 h to 4 h + 3 and 8 + 4 h to 11 + 4 h of
//     column m of the block: the keys whose weights that half of the wave has
//     after the scores.
//
// Measured: 2048 causal queries of 32 heads of 128 over 2048 keys, 34.4 GFLOP, in
// 91-100 us. Its products (six of fp4 by fp6, 1.5 times bf16's, and three of bf16)
// are 2.25 times that, 57 us at a large bf16 product's rate; the exponentials, the
// weights' split and the layout of the next tile share the time with them from
// the CU's other workgroup, and the row tile of 32 key tiles, about 2 us each, is what the
// last CU waits for. (The next step's exponentials put between the products by
// hand 5 us more, by scheduling groups 7; the tiles laid out once for all row
// tiles and copied to LDS 2 less here, and more for fewer rows; row tiles split
// into chunks 25 more.)
template <int NB>
struct PromptCfg {
    static constexpr int kBlock = 32 * 16 + 16;
    static constexpr int kWords = (NB + 3) / 4;  // of a key's scale bytes
    static constexpr int kKHalf = NB * kBlock + 128 * kWords;  // codes, scales
    static constexpr int kVHalf = 2 * NB * 1024;
    static constexpr int kBytes = 2 * (kKHalf + kVHalf);  // of a tile
    // A wave's rows of q or of the output pass through LDS, 16 bytes apart in
    // the banks, so that memory is read and written along the rows.
    static constexpr int kRow = 32 * NB + 4;  // floats
    static constexpr int kLowBytes = QPlanes<NB>::kLow ? 3 * QPlanes<NB>::kSteps * kPlaneBytes : 0;  // a wave
    static constexpr int kLoop = 2 * kBytes + kPromptWaves * kLowBytes, kRows = kPromptWaves * 32 * kRow * 4;
    static constexpr int kLds = kLoop > kRows ? kLoop : kRows;
};

// The planes of Q of 32 rows as the weights' kernel takes them: [step][plane]
// kPlaneBytes, then the scale bytes [step][lane] 8 bytes.
template <int NB>
struct SumCfg {
    static constexpr int kSteps = (NB + 1) / 2;
    static constexpr int kBytes = (kSteps * (kQPlanes * kPlaneBytes + 512) + 1023) / 1024 * 1024;
};

template <int NB>
__device__ __forceinline__ void keep_planes(const Mx4Attn& a, int b, int kvh, int tile, const QPlanes<NB>& q) {
    const int lane = threadIdx.x & 63;
    char* to = a.planes + ((static_cast<uint64_t>(b) * a.kv_heads + kvh) * a.planes_ld + tile) * SumCfg<NB>::kBytes;
#pragma unroll
    for (int s = 0; s < QPlanes<NB>::kSteps; ++s) {
#pragma unroll
        for (int n = 0; n < kQPlanes; ++n) store_plane(to + (s * kQPlanes + n) * kPlaneBytes + lane * 16, q.f[s][n]);
        *reinterpret_cast<uint2*>(to + QPlanes<NB>::kSteps * kQPlanes * kPlaneBytes + s * 512 + lane * 8) = uint2{q.scale[s][0], q.scale[s][1]};
    }
}

// What a thread carries from memory to LDS: a unit of each store with its scales.
template <int NB>
struct Carry {
    Mx4Unit<NB> k, ks, v, vs;
};

template <int NB>
__device__ __forceinline__ void load_carry(const Mx4Attn& a, int b, int kvh, int t, int kg, int n, Carry<NB>& c) {
    const uint8_t* ks = a.k + b * a.k_bs;
    const uint8_t* vs = a.v + b * a.v_bs;
    const uint64_t g = static_cast<uint64_t>(kvh) * a.groups + min(t * 16 + kg, (a.kv - 1) / 4);
    c.k = mhip::mx4_load<NB>(reinterpret_cast<const uint32_t*>(ks) + (g * 16 + n) * NB);
    c.ks = mhip::mx4_load<NB>(reinterpret_cast<const uint32_t*>(ks + a.code_bytes) + g * NB);
    c.v = mhip::mx4_load<NB>(reinterpret_cast<const uint32_t*>(vs) + (g * 16 + n) * NB);
    c.vs = mhip::mx4_load<NB>(reinterpret_cast<const uint32_t*>(vs + a.code_bytes) + g * NB);
}
template <int CTRL>
__device__ __forceinline__ uint32_t quad(uint32_t x) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xF, 0xF, true));
}

// K of a tile: group kg of four keys, unit n.
template <int NB>
__device__ __forceinline__ void store_keys(const Carry<NB>& c, char* lds, int kg, int n) {
    using Cfg = PromptCfg<NB>;
    const int half = kg >> 3, j = kg & 7, lane4 = n & 3;
    char* kd = lds + half * Cfg::kKHalf;
    const uint32_t sel1 = lane4 & 1 ? 0x03070105u : 0x06020400u, sel2 = lane4 & 2 ? 0x03020706u : 0x05040100u;
#pragma unroll
    for (int w = 0; w < NB; ++w) {
        const uint32_t x = __builtin_amdgcn_perm(quad<0xB1>(c.k.w[w]), c.k.w[w], sel1);  // lane ^ 1
        const uint32_t y = __builtin_amdgcn_perm(quad<0x4E>(x), x, sel2);                // lane ^ 2
        const int at = 4 * w + lane4, i = at / NB, p = at % NB;
        *reinterpret_cast<uint32_t*>(kd + p * Cfg::kBlock + (4 * j + i) * 16 + (n & ~3)) = y;
    }
#pragma unroll
    for (int w = 0; w < Cfg::kWords; ++w) {
        uint32_t s = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int p = 4 * w + e;
            s |= (p < NB ? c.ks.w[p < NB ? p : 0] >> (8 * lane4) & 255u : 127u) << (8 * e);
        }
        if (n < 4) *reinterpret_cast<uint32_t*>(kd + NB * Cfg::kBlock + w * 128 + (4 * j + n) * 4) = s;
    }
}

// `nan`: a tile's keys of each block whose value is no number, a bit a key.
// Those values go to LDS as zeros; the rows that admit the key get their NaN
// from the bits (a weight of 0 times NaN would reach the others too).
template <int NB>
__device__ __forceinline__ void take_nan(Carry<NB>& c, uint32_t (*nan)[2], int kg, int n) {
    const int half = kg >> 3, j = kg & 7;
    uint32_t bad = 0;
#pragma unroll
    for (int p = 0; p < NB; ++p) bad |= bytes_255(c.vs.w[p]);
    if (bad) {
#pragma unroll
        for (int p = 0; p < NB; ++p) {
            const uint32_t ff = bytes_255(c.vs.w[p]);
            c.vs.w[p] &= ~whole_bytes(ff);
            if (n == 0 && ff) atomicOr(&nan[p][half], byte_bits(ff) << (4 * j));
        }
    }
}

// V of a tile.
template <int NB>
__device__ __forceinline__ void store_values(const Carry<NB>& c, char* lds, int kg, int n) {
    using Cfg = PromptCfg<NB>;
    const int half = kg >> 3, j = kg & 7;
    char* vd = lds + 2 * Cfg::kKHalf + half * Cfg::kVHalf + ((j / 4) * NB * 64 + (j & 1) * 32 + n) * 16 + (j & 2) * 4;
#pragma unroll
    for (int p = 0; p < NB; ++p) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = i * NB + p;
            w[i] = bits(mhip::mx4_bf16(c.v.w[at / 4], mhip::mx4_scale(c.vs.w[p], i), at % 4));
        }
        const uint2 lo = {__builtin_amdgcn_perm(w[1], w[0], 0x05040100u), __builtin_amdgcn_perm(w[3], w[2], 0x05040100u)};
        const uint2 hi = {__builtin_amdgcn_perm(w[1], w[0], 0x07060302u), __builtin_amdgcn_perm(w[3], w[2], 0x07060302u)};
        *reinterpret_cast<uint2*>(vd + p * 1024) = lo;
        *reinterpret_cast<uint2*>(vd + p * 1024 + 256) = hi;
    }
}

__device__ __forceinline__ Frag lds_frag(const char* p) {
    Frag f;
    __builtin_memcpy(&f, __builtin_assume_aligned(p, 16), 16);
    return f;
}

// S^T of a tile's 64 keys by the wave's 32 rows: st[kk][r] is key 32 kk + 8 (r /
// 4) + 4 h + r % 4 of row lane % 32.
template <int NB>
__device__ __forceinline__ void tile_scores(const char* kt, const QPlanes<NB>& q, const char* low, int m, int h, f32x16 (&st)[2]) {
    using Cfg = PromptCfg<NB>;
    const char* k0 = kt;
    const char* k1 = kt + Cfg::kKHalf;
    uint32_t scale0[Cfg::kWords], scale1[Cfg::kWords];
#pragma unroll
    for (int w = 0; w < Cfg::kWords; ++w) {
        scale0[w] = *reinterpret_cast<const uint32_t*>(k0 + NB * Cfg::kBlock + w * 128 + m * 4) >> (8 * h);
        scale1[w] = *reinterpret_cast<const uint32_t*>(k1 + NB * Cfg::kBlock + w * 128 + m * 4) >> (8 * h);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) st[0][e] = st[1][e] = 0.0f;
    constexpr int kSteps = QPlanes<NB>::kSteps;
    Frag k[kSteps][2];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int at = min(2 * i + h, NB - 1) * Cfg::kBlock + m * 16;
        k[i][0] = lds_frag(k0 + at);
        k[i][1] = lds_frag(k1 + at);
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        if (i % 2 == 0)
            score_step<0>(k[i][0], k[i][1], scale0[i / 2], scale1[i / 2], q, i, low, st);
        else
            score_step<2>(k[i][0], k[i][1], scale0[i / 2], scale1[i / 2], q, i, low, st);
    }
}

// 16 bytes a lane from memory to 1024 bytes of LDS, whose address is the
// wave's. As an instruction of its own: the compiler has every read of LDS wait
// for the builtin's, here the planes in use for the next ones. (m0 is reserved:
// the compiler keeps nothing in it over other instructions.) Its caller waits
// for vmcnt before the barrier that gives the bytes to the other waves.
__device__ __forceinline__ void copy_to_lds(const char* from, char* to) {
    const uint32_t at = __builtin_amdgcn_readfirstlane(
        static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)to)));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from) : "memory");
}

// The words of a tile's NaN bits together.
__device__ __forceinline__ uint32_t any_nan(const uint32_t* flags, int words) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < words; ++i) any |= flags[i];
    return any;
}

// A prompt's place in the grid: the heaviest (latest) row tiles first over all
// heads, then the chunks of a row tile, `chunk_tiles` tiles each. Of a grid of
// two workgroups a CU the second halves go up from the lightest, so that a CU
// gets one with the other.
struct PromptPlace {
    int b, kvh, tile, chunk;
    int row0, row_last;
    int t0, t1;     // the chunk's tiles
    int chunks;     // of this row tile
};
__device__ __forceinline__ PromptPlace prompt_place(const Mx4Attn& a, int block) {
    PromptPlace w;
    const int pairs = a.kv_heads * a.batch;
    const int unit = block / pairs, pair = block - unit * pairs;
    const int rank = a.chunks > 1 ? unit / a.chunks : unit;
    w.chunk = a.chunks > 1 ? unit - rank * a.chunks : 0;
    w.tile = rank < a.heavy_ranks ? a.row_tiles - 1 - rank : rank - a.heavy_ranks;
    w.b = pair / a.kv_heads;
    w.kvh = pair - w.b * a.kv_heads;
    w.row0 = w.tile * kPromptRows;
    w.row_last = min(w.row0 + kPromptRows, a.rows) - 1;
    const int begin = row_keys(a, a.kv, w.row0).lo / 64, end = (row_keys(a, a.kv, w.row_last).hi + 63) / 64;
    w.chunks = a.chunks > 1 ? (end - begin + a.chunk_tiles - 1) / a.chunk_tiles : 1;
    w.t0 = begin + w.chunk * a.chunk_tiles;
    w.t1 = a.chunks > 1 ? min(w.t0 + a.chunk_tiles, end) : end;
    return w;
}

template <int NB>
__global__ __launch_bounds__(64 * kPromptWaves, NB > 4 ? 1 : 2) void mx4_prompt_kernel(Mx4Attn a) {
    using Cfg = PromptCfg<NB>;
    constexpr int DP = 32 * NB;
    __shared__ __attribute__((aligned(16))) char lds[Cfg::kLds];
    __shared__ uint32_t nan[3][NB][2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = lane & 31, h = lane >> 5, kg = tid >> 4, n = tid & 15;
    const PromptPlace at = prompt_place(a, blockIdx.x);
    if (at.chunk >= at.chunks) return;
    const int b = at.b, kvh = at.kvh, t0 = at.t0, t1 = at.t1;

    const int wrow0 = min(at.row0 + wave * 32, a.rows - 1), wrow_last = min(wrow0 + 31, a.rows - 1);
    const int row = min(at.row0 + wave * 32 + q, a.rows - 1);
    const bool wave_live = at.row0 + wave * 32 < a.rows;
    const Keys mine = row_keys(a, a.kv, row);
    const Keys whead = row_keys(a, a.kv, wrow0), wtail = row_keys(a, a.kv, wrow_last);

    Carry<NB> carry;
    load_carry<NB>(a, b, kvh, t0, kg, n, carry);
    float* wrows = reinterpret_cast<float*>(lds) + wave * 32 * Cfg::kRow;
    for (int u = lane; u < 8 * DP; u += 64) {
        const int r = u / (DP / 4), col = u % (DP / 4) * 4;
        const int from = min(at.row0 + wave * 32 + r, a.rows - 1);
        *reinterpret_cast<f32x4*>(wrows + r * Cfg::kRow + col) = load_q4(a, a.q + b * a.q_bs + row_at(a, kvh, from), col);
    }
    if (tid < 6 * NB) (&nan[0][0][0])[tid] = 0;
    __syncthreads();
    QPlanes<NB> qp;
    make_q_planes<NB>(wrows + q * Cfg::kRow, h, qp);
    if (a.planes && at.chunk == 0 && wave_live) keep_planes<NB>(a, b, kvh, at.row0 / 32 + wave, qp);
    __syncthreads();
    char* low = lds + 2 * Cfg::kBytes + wave * Cfg::kLowBytes + lane * 16;
    if constexpr (QPlanes<NB>::kLow)
#pragma unroll
        for (int s = 0; s < QPlanes<NB>::kSteps; ++s)
#pragma unroll
            for (int n = 0; n < 3; ++n) store_plane(low + (3 * s + n) * kPlaneBytes, qp.f[s][3 + n]);
    take_nan<NB>(carry, nan[0], kg, n);
    store_keys<NB>(carry, lds, kg, n);
    store_values<NB>(carry, lds, kg, n);
    load_carry<NB>(a, b, kvh, t0 + 1, kg, n, carry);

    f32x16 o[NB];
#pragma unroll
    for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[c][e] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    int slot = 0;  // (t - t0) % 3
    for (int t = t0; t < t1; ++t) {
        const int base = 64 * t, next = slot == 2 ? 0 : slot + 1, after = next == 2 ? 0 : next + 1;
        __syncthreads();
        if (tid < 2 * NB) (&nan[after][0][0])[tid] = 0;
        const char* kt = lds + ((t - t0) & 1) * Cfg::kBytes;
        const char* vt = kt + 2 * Cfg::kKHalf;
        char* to = lds + ((t + 1 - t0) & 1) * Cfg::kBytes;
        if (!(wave_live && base < wtail.hi && base + 64 > whead.lo)) {
            take_nan<NB>(carry, nan[next], kg, n);
            store_keys<NB>(carry, to, kg, n);
            store_values<NB>(carry, to, kg, n);
            load_carry<NB>(a, b, kvh, t + 2, kg, n, carry);
        } else {
            f32x16 st[2];
            const uint32_t no_number = any_nan(&nan[slot][0][0], 2 * NB);
            tile_scores<NB>(kt, qp, low, q, h, st);
            take_nan<NB>(carry, nan[next], kg, n);
            store_keys<NB>(carry, to, kg, n);
            store_values<NB>(carry, to, kg, n);
            load_carry<NB>(a, b, kvh, t + 2, kg, n, carry);
            if (base < wtail.lo || base + 64 > whead.hi) {
                asm volatile("");  // a branch: 96 instructions that few tiles need
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int key = base + 32 * kk + 8 * (e / 4) + 4 * h + e % 4;
                        if (outside(mine, key)) st[kk][e] = -INFINITY;
                    }
            }
            float top = -INFINITY;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, st[kk][e]);
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            // The maximum moves only when a score passes it by 2^8: weights of up
            // to 2^8 are as exact, and few tiles then rescale the sums.
            top *= a.c;
            if (__ballot(top > m + kLag) != 0) {
                const float m_new = fmaxf(m, top);
                const float alpha = __builtin_amdgcn_exp2f(m - (m_new == -INFINITY ? 0.0f : m_new));
                m = m_new;
                l *= alpha;
#pragma unroll
                for (int c = 0; c < NB; ++c)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[c][e] *= alpha;
            }
            const float m_use = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float p[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[kk][8 * u + e], a.c, -m_use));
                        l += p[e];
                    }
                    Frag w[3];
                    split8(p, w);
#pragma unroll
                    for (int c = 0; c < NB; ++c) {
                        const Frag f = lds_frag(vt + kk * Cfg::kVHalf + ((u * NB + c) * 64 + lane) * 16);
                        o[c] = mfma32(f, w[2], o[c]);
                        o[c] = mfma32(f, w[1], o[c]);
                        o[c] = mfma32(f, w[0], o[c]);
                    }
                }
            if (__builtin_amdgcn_readfirstlane(no_number) != 0) {
                asm volatile("");  // a branch
#pragma unroll
                for (int c = 0; c < NB; ++c) {
                    const uint32_t* flags = nan[slot][c];
                    const uint64_t bad = static_cast<uint64_t>(flags[1]) << 32 | flags[0];
                    const int lo = min(max(mine.lo - base, 0), 64), hi = min(max(mine.hi - base, 0), 64);
                    const uint64_t mask = (hi == 64 ? ~0ull : (1ull << hi) - 1) & ~(lo == 64 ? ~0ull : (1ull << lo) - 1);
                    if (bad & mask)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[c][e] = NAN;
                }
            }
        }
        slot = next;
    }
    l += __shfl_xor(l, 32, 64);
    // The outputs of several chunks as they are, else divided, along the rows.
    const float inv = 1.0f / l, f = at.chunks > 1 ? 1.0f : inv;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            *reinterpret_cast<f32x4*>(wrows + q * Cfg::kRow + 32 * c + 8 * e + 4 * h) =
                f32x4{o[c][4 * e] * f, o[c][4 * e + 1] * f, o[c][4 * e + 2] * f, o[c][4 * e + 3] * f};
    __syncthreads();
    const uint64_t pair = static_cast<uint64_t>(b) * a.kv_heads + kvh;
    const uint64_t rec = ((pair * a.row_tiles + at.tile) * a.chunks + at.chunk) * kPromptRows + wave * 32;
    const int wlive = min(a.rows - at.row0 - wave * 32, 32);
    for (int u = lane; u < wlive * (DP / 4); u += 64) {
        const int r = u / (DP / 4), col = u % (DP / 4) * 4;
        const f32x4 x = *reinterpret_cast<const f32x4*>(wrows + r * Cfg::kRow + col);
        if (at.chunks > 1)
            *reinterpret_cast<f32x4*>(a.part_o + (rec + r) * DP + col) = x;
        else
            store_out(a, b, kvh, at.row0 + wave * 32 + r, col, x);
    }
    if (h == 0 && q < wlive) {
        if (at.chunks > 1) {
            *reinterpret_cast<f32x2*>(a.part_ml + (rec + q) * 2) = f32x2{m, l};
        } else if (a.stats) {
            float* to = a.stats + (pair * a.rows + row) * 2;
            to[0] = m == -INFINITY ? 0.0f : m;
            to[1] = inv;
        }
    }
}

// The chunks' records of the rows whose tile has several, in their order, each
// weighted by 2 to its maximum less the largest. Four columns a thread.
template <int NB>
__global__ __launch_bounds__(256) void mx4_prompt_merge_kernel(Mx4Attn a) {
    constexpr int DP = 32 * NB, kCells = DP / 4, kRows = 256 / kCells;
    if (static_cast<int>(threadIdx.x) >= kRows * kCells) return;
    const int row = blockIdx.x * kRows + threadIdx.x / kCells, col = threadIdx.x % kCells * 4;
    const int kvh = blockIdx.y, b = blockIdx.z;
    if (row >= a.rows) return;
    const int tile = row / kPromptRows, row_last = min((tile + 1) * kPromptRows, a.rows) - 1;
    const int begin = row_keys(a, a.kv, tile * kPromptRows).lo / 64, end = (row_keys(a, a.kv, row_last).hi + 63) / 64;
    const int chunks = (end - begin + a.chunk_tiles - 1) / a.chunk_tiles;
    if (chunks == 1) return;
    const uint64_t pair = static_cast<uint64_t>(b) * a.kv_heads + kvh;
    const uint64_t rec = (pair * a.row_tiles + tile) * a.chunks * kPromptRows + row % kPromptRows;
    float top = -INFINITY;
    for (int c = 0; c < chunks; ++c) top = fmaxf(top, a.part_ml[(rec + c * kPromptRows) * 2]);
    const float m = top == -INFINITY ? 0.0f : top;
    float l = 0.0f;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c = 0; c < chunks; ++c) {
        const uint64_t r = rec + c * kPromptRows;
        const f32x2 ml = *reinterpret_cast<const f32x2*>(a.part_ml + r * 2);
        const float f = __builtin_amdgcn_exp2f(ml.x - m);
        l += ml.y * f;
        sum += *reinterpret_cast<const f32x4*>(a.part_o + r * DP + col) * f;
    }
    const float inv = 1.0f / l;
    store_out(a, b, kvh, row, col, sum * inv);
    if (a.stats && col == 0) {
        a.stats[(pair * a.rows + row) * 2] = m;
        a.stats[(pair * a.rows + row) * 2 + 1] = inv;
    }
}

// The attention each key received, from the scores that the rows kernel kept
// (one row tile): weights_out = weights + the sum over the rows of p. Four keys
// a thread. 4 us beside the attention's 17 for 4 sequences of 8 KV heads over
// 8191 keys: a launch and two loads in turn.
__global__ __launch_bounds__(256) void mx4_kept_weights_kernel(Mx4Attn a, const float* __restrict__ weights,
                                                               float* weights_out, uint64_t stride) {
    const int kv = a.kv + (a.advance ? static_cast<int>(*a.advance) : 0);
    const int key = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (key >= kv) return;
    const uint64_t bh = static_cast<uint64_t>(blockIdx.z) * a.kv_heads + blockIdx.y;
    const float* st = a.stats + bh * a.rows * 2;
    float sum[4] = {};
    for (int row = 0; row < a.rows; ++row) {
        const Keys in = row_keys(a, kv, row);
        if (key + 3 < in.lo || key >= in.hi) continue;
        const f32x4 s = *reinterpret_cast<const f32x4*>(a.kept + (bh * a.rows + row) * a.kept_ld + key);
        const float m = st[2 * row], inv = st[2 * row + 1];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x], a.c, -m)) * inv;
            if (key + x >= in.lo && key + x < in.hi) sum[x] += p;
        }
    }
    const uint64_t at = bh * stride + key;
#pragma unroll
    for (int x = 0; x < 4; ++x)
        if (key + x < kv) weights_out[at + x] = (weights ? weights[at + x] : 0.0f) + sum[x];
}

// The planes of Q for the weights' kernel where the rows kernel took the call (the
// prompts' kernel keeps its own): a wave 32 rows, by way of LDS. 13 us for 1021
// queries of 32 heads of 128, 17 MB read and 20 written.
template <int NB>
__global__ __launch_bounds__(64) void mx4_planes_kernel(Mx4Attn a) {
    constexpr int DP = 32 * NB, kRow = PromptCfg<NB>::kRow;
    __shared__ float rows[32 * kRow];
    const int lane = threadIdx.x, tile = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    for (int u = lane; u < 8 * DP; u += 64) {
        const int r = u / (DP / 4), col = u % (DP / 4) * 4;
        const int from = min(tile * 32 + r, a.rows - 1);
        *reinterpret_cast<f32x4*>(rows + r * kRow + col) = load_q4(a, a.q + b * a.q_bs + row_at(a, kvh, from), col);
    }
    __syncthreads();
    QPlanes<NB> q;
    make_q_planes<NB>(rows + (lane & 31) * kRow, lane >> 5, q);
    keep_planes<NB>(a, b, kvh, tile, q);
}

// The attention each key received from any number of rows, the scores taken
// again by the prompts' scaled products from the planes of Q and the statistics
// that the attention left: a wave holds 64 keys and walks the tiles of 32 rows
// that admit one of the workgroup's (its share of them, of `chunks`), whose
// planes the four waves share in LDS. The rows are the products' columns: a lane's
// sums are its keys' over one column, and the columns are added up at the end, in
// a fixed order; so are the chunks' sums, by mx4_sum_weights_kernel. 20 us and 5 for the
// sums beside an attention of 54 (1021 queries of 32 heads of 128 over as many
// keys). A KV head's workgroups are `pairs` apart in the grid, on one XCD where
// the heads are a multiple of eight, whose L2 then holds the head's planes (37 us for
// 32 with neighbours in the grid); the last 12 were K's codes read by bytes and
// the lanes' sums added up one key at a time.
constexpr int kSumKeys = 64 * kPromptWaves, kSumRows = 8;
template <int NB>
__global__ __launch_bounds__(64 * kPromptWaves) void mx4_weights_kernel(Mx4Attn a, const float* __restrict__ weights,
                                                                               float* weights_out, uint64_t stride, int chunks,
                                                                        float* part, uint64_t part_ld) {
    using Cfg = SumCfg<NB>;
    if (a.advance) a.kv += static_cast<int>(*a.advance);
    constexpr int kSteps = Cfg::kSteps;
    __shared__ __attribute__((aligned(16))) char lds[2][Cfg::kBytes];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = lane & 31, h = lane >> 5;
    const int pairs = a.kv_heads * a.batch, unit = blockIdx.x / pairs, pair = blockIdx.x - unit * pairs;
    const int b = pair / a.kv_heads, kvh = pair - b * a.kv_heads;
    const int block = unit / chunks, chunk = unit - block * chunks;
    const int first = block * kSumKeys, base = first + wave * 64;
    if (first >= a.kv) return;

    // The rows whose queries admit a key of the workgroup, the chunk's share.
    const int off = a.kv - a.seq, last_key = min(first + kSumKeys, a.kv) - 1;
    const int i0 = a.causal ? max(0, first - off) : 0;
    const int64_t past = static_cast<int64_t>(last_key) - off + a.window;  // a window's last query, and one
    const int i1 = a.window > 0 ? static_cast<int>(max(min(static_cast<int64_t>(a.seq), past), static_cast<int64_t>(0))) : a.seq;
    const int begin = i0 * a.group / 32, end = max((i1 * a.group + 31) / 32, begin), per = (end - begin + chunks - 1) / chunks;
    const int r0 = min(begin + chunk * per, end), r1 = min(r0 + per, end);
    const char* planes = a.planes + static_cast<uint64_t>(pair) * a.planes_ld * Cfg::kBytes;
    auto fetch = [&](int t) {
        const char* from = planes + static_cast<uint64_t>(t) * Cfg::kBytes;
#pragma unroll
        for (int i = 0; i < (Cfg::kBytes / 1024 + kPromptWaves - 1) / kPromptWaves; ++i) {
            const int p = i * kPromptWaves + wave;
            if (p < Cfg::kBytes / 1024) copy_to_lds(from + p * 1024 + lane * 16, lds[(t - r0) & 1] + p * 1024);
        }
    };
    if (r0 < r1) fetch(r0);

    // K, halves of 32 keys: lane (key, h), step s: block 2 s + h, 16 bytes, one of
    // each unit.
    Frag k[2][kSteps];
    uint32_t kscale[2][(kSteps + 1) / 2] = {};
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
        const uint8_t* ks = a.k + b * a.k_bs;
        const int key = min(base + 32 * kk + m, a.kv - 1);
        const uint64_t g = static_cast<uint64_t>(kvh) * a.groups + key / 4;
        const uint8_t* unit = ks + g * 64 * NB + (key % 4) * NB;
        const uint8_t* sc = ks + a.code_bytes + g * 4 * NB + key % 4;
        uint32_t four[16];  // heads of four blocks: a key's four bytes of each unit
        if constexpr (NB == 4)
#pragma unroll
            for (int n = 0; n < 16; ++n) four[n] = reinterpret_cast<const uint32_t*>(unit)[4 * n];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int p = min(2 * s + h, NB - 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t w = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (NB == 4)
                        w |= (four[4 * i + e] >> (8 * p) & 255u) << (8 * e);
                    else
                        w |= static_cast<uint32_t>(unit[(4 * i + e) * 4 * NB + p]) << (8 * e);
                }
                k[kk][s].u[i] = w;
            }
            kscale[kk][s / 2] |= (2 * s + h < NB ? static_cast<uint32_t>(sc[4 * p]) : 127u) << (16 * (s % 2));
        }
    }
    const float* stats = a.stats + static_cast<uint64_t>(pair) * a.rows * 2;
    float sum[2][16] = {};  // [half of 32 keys][register of a product]
    auto row_stats = [&](int t) { return *reinterpret_cast<const f32x2*>(stats + 2 * min(32 * t + m, a.rows - 1)); };
    f32x2 next = row_stats(r0);
    for (int t = r0; t < r1; ++t) {
        // This wave's part of the planes is in LDS, and the tile's statistics are
        // in registers before the next fetch is under way.
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        f32x2 st = next;
        asm volatile("" : "+v"(st));
        __syncthreads();
        const int row = min(32 * t + m, a.rows - 1), row_last = min(32 * t + 31, a.rows - 1);
        next = row_stats(t + 1);
        if (t + 1 < r1) fetch(t + 1);
        const Keys head = row_keys(a, a.kv, 32 * t), tail = row_keys(a, a.kv, row_last);
        if (head.lo >= base + 64 || tail.hi <= base) continue;
        const char* q = lds[(t - r0) & 1];
        f32x16 c[2];
#pragma unroll
        for (int e = 0; e < 16; ++e) c[0][e] = c[1][e] = 0.0f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const uint2 scale = *reinterpret_cast<const uint2*>(q + kSteps * kQPlanes * kPlaneBytes + s * 512 + lane * 8);
            const uint32_t s0 = kscale[0][s / 2] >> (16 * (s % 2)), s1 = kscale[1][s / 2] >> (16 * (s % 2));
            auto both = [&](auto opq, int n, uint32_t qs) {
                const u32x6 f = load_plane(q + (s * kQPlanes + n) * kPlaneBytes + lane * 16);
                c[0] = scaled_product<0, decltype(opq)::value>(k[0][s], s0, f, qs, c[0]);
                c[1] = scaled_product<0, decltype(opq)::value>(k[1][s], s1, f, qs, c[1]);
            };
            both(std::integral_constant<int, 1>{}, 5, scale.y);
            both(std::integral_constant<int, 0>{}, 4, scale.y);
            both(std::integral_constant<int, 3>{}, 3, scale.x);
            both(std::integral_constant<int, 2>{}, 2, scale.x);
            both(std::integral_constant<int, 1>{}, 1, scale.x);
            both(std::integral_constant<int, 0>{}, 0, scale.x);
        }
        if (tail.lo <= base && head.hi >= base + 64 && 32 * t + 31 < a.rows) {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    sum[kk][e] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(c[kk][e], a.c, -st.x)), st.y, sum[kk][e]);
        } else {
            Keys mine = row_keys(a, a.kv, row);
            if (32 * t + m >= a.rows) mine.hi = mine.lo;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(c[kk][e], a.c, -st.x));
                    if (!outside(mine, base + 32 * kk + 8 * (e / 4) + 4 * h + e % 4)) sum[kk][e] = __builtin_fmaf(p, st.y, sum[kk][e]);
                }
        }
    }
    // 32 keys' sums over 32 lanes: a lane passes on the half that is not its own,
    // and has key m of them at the end.
    float* v = &sum[0][0];
#pragma unroll
    for (int d = 16; d > 0; d /= 2)
#pragma unroll
        for (int j = 0; j < d; ++j) {
            const float keep = m & d ? v[j + d] : v[j], pass = m & d ? v[j] : v[j + d];
            v[j] = keep + __shfl_xor(pass, d, 64);
        }
    const int key = base + 32 * (m / 16) + 8 * (m % 16 / 4) + 4 * h + m % 4;
    if (key >= a.kv) return;
    if (chunks > 1) {
        part[(static_cast<uint64_t>(pair) * chunks + chunk) * part_ld + key] = v[0];
    } else {
        const uint64_t at = static_cast<uint64_t>(pair) * stride + key;
        weights_out[at] = (weights ? weights[at] : 0.0f) + v[0];
    }
}

// The chunks' sums of a key, in their order.
__global__ __launch_bounds__(256) void mx4_sum_weights_kernel(Mx4Attn a, const float* __restrict__ part, uint64_t part_ld, int chunks,
                                                              const float* __restrict__ weights, float* weights_out, uint64_t stride) {
    const int key = blockIdx.x * 256 + threadIdx.x;
    if (key >= a.kv + (a.advance ? static_cast<int>(*a.advance) : 0)) return;
    const uint64_t pair = static_cast<uint64_t>(blockIdx.z) * a.kv_heads + blockIdx.y;
    float sum = 0.0f;
#pragma unroll 4
    for (int c = 0; c < chunks; ++c) sum += part[(pair * chunks + c) * part_ld + key];
    weights_out[pair * stride + key] = (weights ? weights[pair * stride + key] : 0.0f) + sum;
}

struct KeyTiles {
    uint64_t all = 0, most = 0;
};
// The key tiles that the prompts' row tiles of one KV head see, all together and
// the most of one. (Of very long prompts the first 4096 row tiles: neither the
// choice of a kernel nor a split hangs on the rest.)
KeyTiles key_tiles(const Mx4Attn& a) {
    KeyTiles k;
    for (int row = 0, t = 0; row < a.rows && t < 4096; row += kPromptRows, ++t) {
        const int i0 = row / a.group, i1 = (std::min(row + kPromptRows, a.rows) - 1) / a.group, at = a.kv - a.seq;
        const int lo = a.window > 0 ? std::max(at + i0 - (a.window - 1), 0) : 0, hi = a.causal ? at + i1 + 1 : a.kv;
        const uint64_t n = static_cast<uint64_t>((hi + 63) / 64 - lo / 64);
        k.all += n;
        k.most = std::max(k.most, n);
    }
    return k;
}

// How the weights of more than one row tile are taken: the scratch (planes and
// chunks' sums, 16-byte multiples) and the launches.
struct SumPlan {
    uint64_t keys = 0, key_blocks = 0, chunks = 1, plane_bytes = 0, part_bytes = 0;
};
template <int NB>
SumPlan sum_plan(mhip_ctx* ctx, Mx4Attn& a, uint64_t pairs, uint64_t kv_rows) {
    SumPlan p;
    p.keys = a.advance ? kv_rows : static_cast<uint64_t>(a.kv);
    const uint64_t row_blocks = mhip::ceil_div(a.rows, 32);
    a.planes_ld = row_blocks;
    // Two workgroups for each CU, of at least eight row tiles.
    p.key_blocks = mhip::ceil_div(p.keys, kSumKeys);
    p.chunks = std::max<uint64_t>(1, std::min(mhip::ceil_div(2ull * ctx->compute_units, p.key_blocks * pairs), row_blocks / kSumRows));
    p.plane_bytes = pairs * row_blocks * SumCfg<NB>::kBytes;
    p.part_bytes = p.chunks > 1 ? (pairs * p.chunks * p.keys * sizeof(float) + 15) / 16 * 16 : 0;
    return p;
}
template <int NB>
mhip_status launch_weights(mhip_ctx* ctx, const Mx4Attn& a, uint64_t batch, bool planes, const SumPlan& p, float* part,
                           const float* weights, float* weights_out, uint64_t stride) {
    const dim3 heads(1, static_cast<unsigned>(a.kv_heads), static_cast<unsigned>(batch));
    const uint64_t blocks = p.key_blocks * p.chunks * a.kv_heads * batch;
    if (blocks * kPromptWaves * 64 >= (1ULL << 32)) return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "attention: too many rows");
    if (!planes) mhip::launch(ctx, mx4_planes_kernel<NB>, dim3(static_cast<unsigned>(a.planes_ld), heads.y, heads.z), dim3(64), 0, a);
    mhip::launch(ctx, mx4_weights_kernel<NB>, dim3(static_cast<unsigned>(blocks)),
                 dim3(64 * kPromptWaves), 0, a, weights, weights_out, stride, static_cast<int>(p.chunks), part, p.keys);
    if (p.chunks > 1)
        mhip::launch(ctx, mx4_sum_weights_kernel, dim3(static_cast<unsigned>(mhip::ceil_div(p.keys, 256)), heads.y, heads.z), dim3(256), 0,
                     a, part, p.keys, static_cast<int>(p.chunks), weights, weights_out, stride);
    return mhip::check_launch("attention (4-bit, weights)");
}

template <int NB, bool FEW>
mhip_status launch_rows(mhip_ctx* ctx, Mx4Attn& a, uint64_t batch, const float* weights, float* weights_out,
                        uint64_t stride, uint64_t kv_rows) {
    a.row_tiles = static_cast<int>(mhip::ceil_div(a.rows, kRowTile<FEW>));
    a.batch = static_cast<int>(batch);
    const uint64_t tiles = batch * a.kv_heads * a.row_tiles;
    // A workgroup for each CU, of at least a strip a wave. (Two on each, with half
    // the chunk: 8 x 4096 keys 19 us for 15, 131073 keys 42 for 33, what the
    // waves' own part and the records cost more than what they hide.)
    uint64_t chunks = mhip::ceil_div(ctx->compute_units, tiles);
    chunks = std::min<uint64_t>({chunks, mhip::ceil_div(kv_rows, 64 * kRowWaves<NB>), kMaxChunks});
    if (tiles > mhip::kMx4Counters) chunks = 1;
    a.chunks = static_cast<int>(chunks);
    const uint64_t records = tiles * chunks * kRowTile<FEW>;
    const uint64_t total_rows = batch * a.kv_heads * static_cast<uint64_t>(a.rows);
    if (a.row_tiles * chunks * kRowWaves<NB> * 64 >= (1ULL << 32))
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "attention: too many rows");
    const bool keep = weights_out && a.row_tiles == 1;
    a.kept_ld = (kv_rows + 63) / 64 * 64;
    const SumPlan sums = weights_out && !keep ? sum_plan<NB>(ctx, a, batch * a.kv_heads, kv_rows) : SumPlan{};
    // Scratch: planes, chunk records, kept scores, chunks' sums, statistics.
    const uint64_t record_bytes = chunks > 1 ? records * (32 * NB + 2) * sizeof(float) : 0;
    const uint64_t kept_bytes = keep ? total_rows * a.kept_ld * sizeof(float) : 0;
    const uint64_t bytes = sums.plane_bytes + record_bytes + kept_bytes + sums.part_bytes + (weights_out ? total_rows * 2 * sizeof(float) : 0);
    float* part = nullptr;
    if (bytes) {
        void* ws = nullptr;
        mhip_status st = mhip::workspace(ctx, bytes, &ws);
        if (st != MHIP_OK) return st;
        char* at = static_cast<char*>(ws);
        a.planes = at;
        a.part_o = reinterpret_cast<float*>(at += sums.plane_bytes);
        a.part_ml = a.part_o + records * (32 * NB);
        a.kept = keep ? reinterpret_cast<float*>(at + record_bytes) : nullptr;
        part = reinterpret_cast<float*>(at += record_bytes + kept_bytes);
        if (weights_out) a.stats = reinterpret_cast<float*>(at + sums.part_bytes);
    }
    a.arrived = ctx->mx4_arrived;
    const dim3 grid(static_cast<unsigned>(a.row_tiles * chunks), static_cast<unsigned>(a.kv_heads), static_cast<unsigned>(batch));
    mhip::launch(ctx, mx4_rows_kernel<NB, FEW>, grid, dim3(64 * kRowWaves<NB>), 0, a);
    mhip_status st = mhip::check_launch("attention (4-bit)");
    if (st != MHIP_OK || !weights_out) return st;
    if (!keep) return launch_weights<NB>(ctx, a, batch, false, sums, part, weights, weights_out, stride);
    const uint64_t keys = a.advance ? kv_rows : static_cast<uint64_t>(a.kv);
    mhip::launch(ctx, mx4_kept_weights_kernel,
                 dim3(static_cast<unsigned>(mhip::ceil_div(keys, 1024)), static_cast<unsigned>(a.kv_heads), static_cast<unsigned>(batch)),
                 dim3(256), 0, a, weights, weights_out, stride);
    return mhip::check_launch("attention (4-bit, weights)");
}

template <int NB>
mhip_status launch_prompt(mhip_ctx* ctx, Mx4Attn& a, uint64_t batch, const float* weights, float* weights_out,
                          uint64_t stride) {
    a.row_tiles = static_cast<int>(mhip::ceil_div(a.rows, kPromptRows));
    a.batch = static_cast<int>(batch);
    const uint64_t pairs = batch * a.kv_heads, tiles = pairs * a.row_tiles;
    const KeyTiles keys = key_tiles(a);
    const uint64_t units = keys.all * pairs, most = keys.most;
    const uint64_t slots = (NB > 4 ? 1ull : 2ull) * ctx->compute_units;
    a.chunks = 1;
    a.chunk_tiles = 0;
    a.heavy_ranks = a.row_tiles;
    if (tiles < ctx->compute_units) {
        const uint64_t len = std::max<uint64_t>(kMinChunk, mhip::ceil_div(units, slots));
        if (len < most) {
            a.chunk_tiles = static_cast<int>(len);
            a.chunks = static_cast<int>(mhip::ceil_div(most, len));
        }
    }
    if (a.chunks == 1 && tiles > ctx->compute_units && tiles <= slots)
        a.heavy_ranks = static_cast<int>(mhip::ceil_div(ctx->compute_units, pairs));
    if (tiles * a.chunks * kPromptWaves * 64 >= (1ULL << 32)) return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "attention: too many rows");
    const uint64_t records = a.chunks > 1 ? tiles * a.chunks * kPromptRows : 0;
    const SumPlan sums = weights_out ? sum_plan<NB>(ctx, a, pairs, a.kv) : SumPlan{};
    const uint64_t record_bytes = records * (32 * NB + 2) * sizeof(float);
    const uint64_t bytes = sums.plane_bytes + record_bytes + sums.part_bytes + (weights_out ? pairs * a.rows * 2 * sizeof(float) : 0);
    float* part = nullptr;
    if (bytes) {
        void* ws = nullptr;
        mhip_status st = mhip::workspace(ctx, bytes, &ws);
        if (st != MHIP_OK) return st;
        char* at = static_cast<char*>(ws);
        a.planes = weights_out ? at : nullptr;
        a.part_o = reinterpret_cast<float*>(at += sums.plane_bytes);
        a.part_ml = a.part_o + records * (32 * NB);
        part = reinterpret_cast<float*>(at += record_bytes);
        if (weights_out) a.stats = reinterpret_cast<float*>(at + sums.part_bytes);
    }
    const dim3 grid(static_cast<unsigned>(tiles * a.chunks)), block(64 * kPromptWaves);
    mhip::launch(ctx, mx4_prompt_kernel<NB>, grid, block, 0, a);
    mhip_status st = mhip::check_launch("attention (4-bit, prompt)");
    const dim3 heads(1, static_cast<unsigned>(a.kv_heads), static_cast<unsigned>(batch));
    if (st == MHIP_OK && a.chunks > 1) {
        mhip::launch(ctx, mx4_prompt_merge_kernel<NB>, dim3(static_cast<unsigned>(mhip::ceil_div(a.rows, 256 / (8 * NB))), heads.y, heads.z),
                     dim3(256), 0, a);
        st = mhip::check_launch("attention (4-bit, prompt merge)");
    }
    if (st != MHIP_OK || !weights_out) return st;
    return launch_weights<NB>(ctx, a, batch, true, sums, part, weights, weights_out, stride);
}

// Which of the two attention kernels is the faster one, in microseconds of time
// that both were measured to take on 256 CUs (2 to 20 % off over rows of 5 to
// 2048 queries and 1000 to 30000 keys, head dimensions 64 to 192): a workgroup
// of the rows kernel 6, and 0.75 a block of 32 columns for each turn of its
// waves over 64 keys; prompts 25 to fill and drain, then 0.46 a block for 128
// rows by 64 keys on one CU. `units`: such row and key tiles in all.
bool prompt_is_faster(const mhip_ctx* ctx, const Mx4Attn& a, uint64_t pairs, uint64_t units, uint64_t nb) {
    const uint64_t row_tiles = mhip::ceil_div(a.rows, 16), waves = nb > 4 ? 4 : 8;
    const double cus = ctx->compute_units, tiles = static_cast<double>(pairs * row_tiles);
    const double chunks = std::max(1.0, std::ceil(cus / tiles));
    const double strips = static_cast<double>(units) * std::min<double>(8, row_tiles) / tiles / chunks;  // of 64 keys a workgroup
    const double rows_us = std::ceil(tiles * chunks / cus) * (6 + 0.75 * nb * std::ceil(strips / waves));
    return 25 + 0.46 * nb * units / cus < rows_us;
}

}  // namespace

extern "C" mhip_status mhip_attention_mx4(mhip_ctx* ctx, const float* q, const void* k_store, const void* v_store,
                                          float* out, const mhip_attention_params* p, const float* weights,
                                          float* weights_out) {
    MHIP_REQUIRE_CTX(ctx);
    if (!p) return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "attention: null params");
    const uint64_t H = p->head_count, Hkv = p->kv_head_count, d = p->head_dimension;
    const uint64_t batch = p->batch ? p->batch : 1;
    if (H == 0 || d == 0 || Hkv == 0)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED,
                          "head_count, kv_head_count, and head_dimension must all be positive");
    if (H % Hkv != 0)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED,
                          "head_count " + std::to_string(H) + " must be an exact multiple of kv_head_count " +
                              std::to_string(Hkv));
    if (p->value_dimension != 0 && p->value_dimension != d)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "attention over 4-bit stores: values have the keys' head dimension");
    const mhip_mx4_store ks = {p->kv_rows, Hkv, d, batch, p->kv_batch_stride};
    const mhip_mx4_store vs = {p->kv_rows, Hkv, d, batch, p->v_batch_stride};
    mhip_status st = mhip::mx4_check(&ks, "attention");
    if (st == MHIP_OK) st = mhip::mx4_check(&vs, "attention");
    if (st != MHIP_OK) return st;
    if (p->window_size == 0)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "window_size must be positive; a zero window admits no keys");
    if (p->window_size > 0 && !p->causal)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "window_size is only defined for causal attention");
    if (p->kv_seq_len > p->kv_rows)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "key_count " + std::to_string(p->kv_seq_len) + " exceeds the " +
                                                      std::to_string(p->kv_rows) + " rows of K/V");
    if (p->seq_len > p->kv_seq_len)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "q sequence length " + std::to_string(p->seq_len) +
                                                      " cannot exceed k/v sequence length " +
                                                      std::to_string(p->kv_seq_len));
    if (!(p->scale <= 0.0f) && !std::isfinite(p->scale))
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "attention scale must be finite and positive");
    if (weights && !weights_out)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "attention: weights without an output for their sums");
    if (p->seq_len == 0 && !weights_out) return MHIP_OK;
    if (p->seq_len == 0)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "attention: no query to add to the weights");
    if (!q || !k_store || !v_store || !out) return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "attention: null buffer");
    if (!mhip::aligned16(k_store) || !mhip::aligned16(v_store))
        return mhip::fail(MHIP_LAYOUT_UNSUPPORTED, "attention: the stores must be 16-byte aligned");
    const uint64_t group = H / Hkv, rows = p->seq_len * group;
    // A grid has fewer than 2^32 threads.
    if (H >= (1ULL << 20) || rows >= (1ULL << 26))
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "attention: too many rows");

    Mx4Attn a{};
    a.q = q;
    a.k = static_cast<const uint8_t*>(k_store);
    a.v = static_cast<const uint8_t*>(v_store);
    a.out = out;
    a.q_ld = H * d;
    a.q_bs = p->q_batch_stride ? p->q_batch_stride : p->seq_len * a.q_ld;
    a.o_bs = p->out_batch_stride ? p->out_batch_stride : p->seq_len * a.q_ld;
    const uint64_t one = mhip::mx4_bytes(p->kv_rows, Hkv, d);
    a.k_bs = p->kv_batch_stride ? p->kv_batch_stride : one;
    a.v_bs = p->v_batch_stride ? p->v_batch_stride : one;
    a.code_bytes = mhip::mx4_code_bytes(p->kv_rows, Hkv, d);
    a.seq = static_cast<int>(p->seq_len);
    a.kv = static_cast<int>(p->kv_seq_len);
    a.rows = static_cast<int>(rows);
    a.heads = static_cast<int>(H);
    a.kv_heads = static_cast<int>(Hkv);
    a.group = static_cast<int>(group);
    a.d = static_cast<int>(d);
    a.groups = static_cast<int>(mhip::mx4_groups(p->kv_rows));
    a.causal = p->causal ? 1 : 0;
    a.window = p->window_size > 0 ? static_cast<int>(std::min<int64_t>(p->window_size, 1LL << 30)) : -1;
    a.vec = d % 4 == 0 && mhip::aligned16(out) && a.o_bs % 4 == 0;
    a.vec_q = d % 4 == 0 && mhip::aligned16(q) && a.q_bs % 4 == 0;
    const float scale = p->scale > 0.0f ? p->scale : 1.0f / std::sqrt(static_cast<float>(d));
    a.c = scale * kLog2e;
    if (p->bounded_key_count) {
        if (p->seq_len == 1)
            a.advance = mhip::advance_ptr(ctx, MHIP_ADVANCE_KEY_COUNT, p->kv_rows - p->kv_seq_len);
        else
            (void)mhip::advance_ptr(ctx, MHIP_ADVANCE_KEY_COUNT, 0);
    }
    const uint64_t plan_rows = p->bounded_key_count ? p->kv_rows : p->kv_seq_len;
    const bool few = a.rows <= kRowTile<true>;
    const uint64_t blocks = mhip::mx4_blocks(d);
    const mhip::CaptureGrowth growth(ctx, true);  // a capture takes the eager call's plan
    // Above six blocks the prompts' sums do not fit the registers.
    if (p->seq_len > 1 && rows > kRowTile<false> && blocks <= 6 && prompt_is_faster(ctx, a, batch * Hkv, key_tiles(a).all * batch * Hkv, blocks)) {
        switch (blocks) {
            case 1: return launch_prompt<1>(ctx, a, batch, weights, weights_out, p->kv_rows);
            case 2: return launch_prompt<2>(ctx, a, batch, weights, weights_out, p->kv_rows);
            case 3: return launch_prompt<3>(ctx, a, batch, weights, weights_out, p->kv_rows);
            case 4: return launch_prompt<4>(ctx, a, batch, weights, weights_out, p->kv_rows);
            case 5: return launch_prompt<5>(ctx, a, batch, weights, weights_out, p->kv_rows);
            default: return launch_prompt<6>(ctx, a, batch, weights, weights_out, p->kv_rows);
        }
    }
    switch (blocks) {
        case 1:
            return few ? launch_rows<1, true>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows)
                       : launch_rows<1, false>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows);
        case 2:
            return few ? launch_rows<2, true>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows)
                       : launch_rows<2, false>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows);
        case 3:
            return few ? launch_rows<3, true>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows)
                       : launch_rows<3, false>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows);
        case 4:
            return few ? launch_rows<4, true>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows)
                       : launch_rows<4, false>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows);
        case 5:
            return few ? launch_rows<5, true>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows)
                       : launch_rows<5, false>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows);
        case 6:
            return few ? launch_rows<6, true>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows)
                       : launch_rows<6, false>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows);
        case 7:
            return few ? launch_rows<7, true>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows)
                       : launch_rows<7, false>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows);
        default:
            return few ? launch_rows<8, true>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows)
                       : launch_rows<8, false>(ctx, a, batch, weights, weights_out, p->kv_rows, plan_rows);
    }
}
