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
// is head r % group of query r / group. A wave takes 16 rows and 64 keys at a
// time (16x16x32 products), and both products are fed from the stores' units
// as they lie in memory. With kg a group of four keys, n a lane of 16 and g one
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
    int row_tiles, chunks;
    float c;                      // scale * log2(e)
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
    for (int b = 0; b < NB; ++b) {
        flags[b] = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t byte = 255u << (8 * i);
                const bool nan = (v.scale[r].w[b] & byte) == byte;
                const bool past = base + 16 * g + 4 * r + i >= hi;
                if (nan || past) v.scale[r].w[b] &= ~byte;
                if (nan && !past) flags[b] |= 1u << (4 * r + i);
            }
        any |= flags[b];
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

constexpr int kWeightWaves = 4;
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
        const bool edge = base < tail.lo || base + 64 > head.hi;
        if (edge) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = base + 16 * g + 4 * r + i;
                    if (key < mine.lo || key >= mine.hi) st[i][r] = -INFINITY;
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

// The attention each key received, from the scores that the rows kernel kept
// (one row tile): weights_out = weights + the sum over the rows of p. Four keys
// a thread.
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

// The same for any number of rows, the scores taken again from the rows'
// statistics. A
// wave takes 64 keys and every row tile that admits one of them.
template <int NB>
__global__ __launch_bounds__(64 * kWeightWaves) void mx4_weights_kernel(Mx4Attn a, const float* __restrict__ weights,
                                                                  float* weights_out, uint64_t stride) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.y, b = blockIdx.z;
    const int kv = a.kv + (a.advance ? static_cast<int>(*a.advance) : 0);
    const int base = (blockIdx.x * kWeightWaves + wave) * 64;
    if (base >= kv) return;
    const uint8_t* ks = a.k + b * a.k_bs;
    const uint64_t head_units = static_cast<uint64_t>(kvh) * a.groups;
    const uint32_t* kc = reinterpret_cast<const uint32_t*>(ks) + head_units * 16 * NB;
    const uint32_t* kx = reinterpret_cast<const uint32_t*>(ks + a.code_bytes) + head_units * NB;
    Strip<NB> k;
    load_k<NB>(kc, kx, base / 4, (kv - 1) / 4, n, g, k);
    float sum[4][4] = {};
    // The first query that admits a key of the strip, and the last.
    int i0 = 0, i1 = a.seq;
    if (a.causal) i0 = max(0, base - (kv - a.seq));
    if (a.window > 0) i1 = static_cast<int>(min(static_cast<int64_t>(a.seq), static_cast<int64_t>(base) + 63 - (kv - a.seq) + a.window));
    const float* stats = a.stats + (static_cast<uint64_t>(b) * a.kv_heads + kvh) * a.rows * 2;
    for (int tile = i0 * a.group / 16; tile * 16 < i1 * a.group; ++tile) {
        const int row = min(tile * 16 + n, a.rows - 1);
        Rows<false> q[NB];
        load_q<NB, false>(a, a.q + b * a.q_bs + row_at(a, kvh, row), g, Plane{}, q);
        f32x4 st[4];
        scores<NB, false>(k, q, st);
        const Keys mine = row_keys(a, kv, row);
        const float m = stats[2 * row], inv = stats[2 * row + 1];
        const bool live = tile * 16 + n < a.rows;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = base + 16 * g + 4 * r + i;
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i][r], a.c, -m)) * inv;
                if (live && key >= mine.lo && key < mine.hi) sum[i][r] += p;
            }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int off = 1; off < 16; off *= 2) sum[i][r] += __shfl_xor(sum[i][r], off, 64);
    if (n == 0) {
        const uint64_t at = (static_cast<uint64_t>(b) * a.kv_heads + kvh) * stride;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = base + 16 * g + 4 * r + i;
                if (key < kv) weights_out[at + key] = (weights ? weights[at + key] : 0.0f) + sum[i][r];
            }
    }
}

template <int NB, bool FEW>
mhip_status launch_rows(mhip_ctx* ctx, Mx4Attn& a, uint64_t batch, const float* weights, float* weights_out,
                        uint64_t stride, uint64_t kv_rows) {
    a.row_tiles = static_cast<int>(mhip::ceil_div(a.rows, kRowTile<FEW>));
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
    if (a.row_tiles * chunks >= (1ULL << 31) || mhip::ceil_div(total_rows, 4) >= (1ULL << 31))
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "attention: too many rows");
    const bool keep = weights_out && a.row_tiles == 1;
    a.kept_ld = (kv_rows + 63) / 64 * 64;
    const uint64_t part_bytes = chunks > 1 ? records * (32 * NB + 2) * sizeof(float) : 0;
    const uint64_t kept_bytes = keep ? total_rows * a.kept_ld * sizeof(float) : 0;
    const uint64_t bytes = part_bytes + kept_bytes + (weights_out ? total_rows * 2 * sizeof(float) : 0);
    if (bytes) {
        void* ws = nullptr;
        mhip_status st = mhip::workspace(ctx, bytes, &ws);
        if (st != MHIP_OK) return st;
        a.part_o = static_cast<float*>(ws);
        a.part_ml = a.part_o + records * (32 * NB);
        a.kept = keep ? reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + part_bytes) : nullptr;
        if (weights_out) a.stats = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + part_bytes + kept_bytes);
    }
    a.arrived = ctx->mx4_arrived;
    const dim3 grid(static_cast<unsigned>(a.row_tiles * chunks), static_cast<unsigned>(a.kv_heads), static_cast<unsigned>(batch));
    mhip::launch(ctx, mx4_rows_kernel<NB, FEW>, grid, dim3(64 * kRowWaves<NB>), 0, a);
    mhip_status st = mhip::check_launch("attention (4-bit)");
    if (st != MHIP_OK || !weights_out) return st;
    const uint64_t keys = a.advance ? kv_rows : static_cast<uint64_t>(a.kv);
    const dim3 heads(1, static_cast<unsigned>(a.kv_heads), static_cast<unsigned>(batch));
    if (keep)
        mhip::launch(ctx, mx4_kept_weights_kernel, dim3(static_cast<unsigned>(mhip::ceil_div(keys, 1024)), heads.y, heads.z),
                     dim3(256), 0, a, weights, weights_out, stride);
    else
        mhip::launch(ctx, mx4_weights_kernel<NB>, dim3(static_cast<unsigned>(mhip::ceil_div(keys, 64 * kWeightWaves)), heads.y, heads.z),
                     dim3(64 * kWeightWaves), 0, a, weights, weights_out, stride);
    return mhip::check_launch("attention (4-bit, weights)");
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
    if (H >= (1ULL << 20) || rows >= (1ULL << 31) - 512)
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
    switch (mhip::mx4_blocks(d)) {
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
