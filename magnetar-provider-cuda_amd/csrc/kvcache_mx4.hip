// The 4-bit store's rows: written (f32 rounded to codes under a power-of-two
// scale a block), read back as f32, and evicted by their accumulated attention
// weights. The format is in mx4.hpp. All of it is bound by memory.
#include "mx4.hpp"

namespace mhip {

mhip_status mx4_check(const mhip_mx4_store* s, const char* what) {
    const std::string at(what);
    if (!s) return fail(MHIP_SHAPE_UNSUPPORTED, at + ": null store shape");
    if (s->kv_heads == 0 || s->head_dimension == 0)
        return fail(MHIP_SHAPE_UNSUPPORTED, at + ": kv_heads and head_dimension must be positive");
    if (s->head_dimension > kMx4MaxDimension)
        return fail(MHIP_SHAPE_UNSUPPORTED, at + ": head dimension " + std::to_string(s->head_dimension) +
                                                " is above " + std::to_string(kMx4MaxDimension));
    if (s->capacity >= (1ULL << 31) - 512 || s->kv_heads >= (1ULL << 16) || s->batch >= (1ULL << 16))
        return fail(MHIP_SHAPE_UNSUPPORTED, at + ": capacity, kv_heads or batch too large");
    if (s->batch_stride % 16 != 0)
        return fail(MHIP_LAYOUT_UNSUPPORTED, at + ": the stride between stores must be a multiple of 16 bytes");
    if (s->batch > 1 && s->batch_stride != 0 &&
        s->batch_stride < mx4_used_bytes(s->capacity, s->kv_heads, s->head_dimension))
        return fail(MHIP_SHAPE_UNSUPPORTED, at + ": the stride between stores is below a store's size");
    return MHIP_OK;
}

}  // namespace mhip

namespace {

using mhip::Mx4Unit;

// A call's store as the kernels see it.
struct StoreArgs {
    uint8_t* base;
    uint64_t stride;      // bytes between sequences' stores
    uint64_t code_bytes;  // of one store, after which its scales begin
    uint32_t groups, heads, d;
};

StoreArgs store_args(const mhip_mx4_store& s, const void* base) {
    StoreArgs a;
    a.base = static_cast<uint8_t*>(const_cast<void*>(base));
    a.stride = s.batch_stride ? s.batch_stride : mhip::mx4_bytes(s.capacity, s.kv_heads, s.head_dimension);
    a.code_bytes = mhip::mx4_code_bytes(s.capacity, s.kv_heads, s.head_dimension);
    a.groups = static_cast<uint32_t>(mhip::mx4_groups(s.capacity));
    a.heads = static_cast<uint32_t>(s.kv_heads);
    a.d = static_cast<uint32_t>(s.head_dimension);
    return a;
}

template <int NB>
__device__ __forceinline__ uint8_t* unit_ptr(const StoreArgs& s, uint32_t b, uint32_t h, uint64_t group, uint32_t n) {
    return s.base + b * s.stride + ((static_cast<uint64_t>(h) * s.groups + group) * 16 + n) * (4 * NB);
}
template <int NB>
__device__ __forceinline__ uint8_t* scale_ptr(const StoreArgs& s, uint32_t b, uint32_t h, uint64_t group) {
    return s.base + b * s.stride + s.code_bytes + (static_cast<uint64_t>(h) * s.groups + group) * (4 * NB);
}

// The exponent byte of a block whose largest magnitude has the bits `top`:
// the smallest power of two under which it rounds to at most 6, the largest
// code, which 7 and above would not. For top = f * 2^x, f in [1, 2), that is
// 2^(x - 2), and twice it from f = 1.75 on: adding 0.25 to f carries into the
// exponent exactly then. Exponents stay in [-120, 125], so that every value is
// a normal bf16 and none overflows (magnitudes from 1.75 * 2^127 on saturate
// at 1.5 * 2^127, blocks below 2^-121 become 0).
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
    if (top >= 0x7F800000u) return mhip::kMx4NaN;
    const int x = static_cast<int>((top + 0x00200000u) >> 23) - 2;
    return static_cast<uint32_t>(min(max(x, 7), 252));
}

// The largest over 16 lanes, in all of them: rotations by 8, 4, 2 and 1.
template <int CTRL>
__device__ __forceinline__ uint32_t max_ror(uint32_t v) {
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, true)));
}
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    return max_ror<0x121>(max_ror<0x122>(max_ror<0x124>(max_ror<0x128>(v))));
}

// 16 lanes take a group of four rows of one head, a lane its unit: 2 NB
// columns of each row, lanes side by side in memory. The block's largest
// magnitude is a maximum over the 16 lanes (as integers: a NaN's bits lie above
// an infinity's, so either marks the block). A group that the call covers
// whole is stored as dwords, one at its ends byte by byte. All four rows' loads
// are out before the first is used, and the maxima stay in registers: 67 MB of
// rows in 14.8 us, 5.1 TB/s read and written (row by row, with maxima by way of
// LDS and 64-bit divisions, 25 us).
template <int NB>
__global__ __launch_bounds__(256) void mx4_write_kernel(const float* __restrict__ rows, StoreArgs s, uint64_t count,
                                                        uint64_t row_offset, const uint64_t* advance,
                                                        uint32_t groups_touched, uint32_t units) {
    const uint32_t u = blockIdx.x * 16 + (threadIdx.x >> 4);
    const uint32_t n = threadIdx.x & 15;
    if (u >= units) return;  // all 16 lanes of a unit row at once
    const uint64_t first = row_offset + (advance ? *advance : 0);
    const uint32_t h = u % s.heads, rest = u / s.heads, b = rest / groups_touched;
    const uint64_t group = first / 4 + rest % groups_touched;
    // The rows [lo, hi) of the group that this call writes.
    const int lo = static_cast<int>(first > group * 4 ? first - group * 4 : 0);
    const uint64_t end = first + count;
    const int hi = end <= group * 4 ? 0 : static_cast<int>(end - group * 4 < 4 ? end - group * 4 : 4);
    const uint64_t width = static_cast<uint64_t>(s.heads) * s.d;

    // Rows that the call does not write are read as one that it does (there is
    // one: groups_touched of a captured call may visit a group without any).
    if (lo >= hi) return;
    float x[4][NB][2];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int from = min(max(r, lo), hi - 1);
        const float* row = rows + (b * count + (group * 4 + from - first)) * width + static_cast<uint64_t>(h) * s.d;
#pragma unroll
        for (int p = 0; p < NB; ++p) {
            const uint32_t c = 32 * p + n;
            const float x0 = row[min(c, s.d - 1)], x1 = row[min(c + 16, s.d - 1)];
            x[r][p][0] = c < s.d ? x0 : 0.0f;
            x[r][p][1] = c + 16 < s.d ? x1 : 0.0f;
        }
    }
    uint32_t code[NB], scale[NB];
#pragma unroll
    for (int p = 0; p < NB; ++p) code[p] = scale[p] = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int p = 0; p < NB; ++p) {
            const float x0 = x[r][p][0], x1 = x[r][p][1];
            const uint32_t top = max16(max(__float_as_uint(x0) & 0x7FFFFFFFu, __float_as_uint(x1) & 0x7FFFFFFFu));
            const uint32_t e = scale_byte(top);
            const uint32_t two = e == mhip::kMx4NaN
                                     ? 0u
                                     : __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x0, x1, __uint_as_float(e << 23), 0);
            const int at = r * NB + p;  // byte of the unit
            code[at / 4] |= (two & 0xFFu) << (8 * (at % 4));
            scale[p] |= e << (8 * r);
        }
    }
    uint8_t* dst = unit_ptr<NB>(s, b, h, group, n);
    uint8_t* sdst = scale_ptr<NB>(s, b, h, group);
    if (lo == 0 && hi == 4) {
        __builtin_memcpy(__builtin_assume_aligned(dst, NB % 4 == 0 ? 16 : NB % 2 == 0 ? 8 : 4), code, 4 * NB);
        if (n == 0) __builtin_memcpy(__builtin_assume_aligned(sdst, NB % 4 == 0 ? 16 : NB % 2 == 0 ? 8 : 4), scale, 4 * NB);
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (r < lo || r >= hi) continue;
#pragma unroll
        for (int p = 0; p < NB; ++p) {
            const int at = r * NB + p;
            dst[at] = static_cast<uint8_t>(code[at / 4] >> (8 * (at % 4)));
            if (n == 0) sdst[4 * p + r] = static_cast<uint8_t>(scale[p] >> (8 * r));
        }
    }
}

// The other way: a lane's unit to its 2 NB columns of the rows asked for. 67 MB
// of rows in 13 us, 5.8 TB/s.
template <int NB>
__global__ __launch_bounds__(256) void mx4_read_kernel(float* __restrict__ rows, StoreArgs s, uint64_t count,
                                                       uint64_t first, uint32_t groups_touched, uint32_t units) {
    const uint32_t u = blockIdx.x * 16 + (threadIdx.x >> 4);
    const uint32_t n = threadIdx.x & 15;
    if (u >= units) return;
    const uint32_t h = u % s.heads, rest = u / s.heads, b = rest / groups_touched;
    const uint64_t group = first / 4 + rest % groups_touched;
    const Mx4Unit<NB> code = mhip::mx4_load<NB>(reinterpret_cast<const uint32_t*>(unit_ptr<NB>(s, b, h, group, n)));
    const Mx4Unit<NB> scale = mhip::mx4_load<NB>(reinterpret_cast<const uint32_t*>(scale_ptr<NB>(s, b, h, group)));
    const uint64_t width = static_cast<uint64_t>(s.heads) * s.d;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const uint64_t row = group * 4 + r;
        if (row < first || row >= first + count) continue;
        float* x = rows + (b * count + (row - first)) * width + static_cast<uint64_t>(h) * s.d;
#pragma unroll
        for (int p = 0; p < NB; ++p) {
            const int at = r * NB + p;
            const mhip::f32x2 v = mhip::mx4_f32(code.w[at / 4], mhip::mx4_scale(scale.w[p], r), at % 4);
            const uint32_t c = 32 * p + n;
            if (c < s.d) x[c] = v.x;
            if (c + 16 < s.d) x[c + 16] = v.y;
        }
    }
}

// ---------------------------------------------------------------------------
// Eviction
// ---------------------------------------------------------------------------

constexpr int kSelectThreads = 1024;

struct SelectArgs {
    const float* weights;  // [batch * heads][weight_stride]
    float* weights_out;    // [batch * heads][out_stride]; may be `weights`
    uint32_t* indices;     // [batch * heads][keep]
    uint64_t weight_stride, out_stride;
    uint32_t count, keep, first, recent, out_rows;
};

// A weight as an integer in its order: NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (!(w >= -INFINITY)) w = -INFINITY;
    if (w == 0.0f) w = 0.0f;
    const uint32_t bits = __float_as_uint(w);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// The sum over the lanes up to this one, in the registers of a wave: shifts
// within rows of 16, then the rows' and the halves' last sums passed on.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t add_dpp(uint32_t v) {
    return v + static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ uint32_t scan64(uint32_t v) {
    v = add_dpp<0x118, 0xF>(add_dpp<0x114, 0xF>(add_dpp<0x112, 0xF>(add_dpp<0x111, 0xF>(v))));  // row_shr
    return add_dpp<0x143, 0xC>(add_dpp<0x142, 0xA>(v));  // row_bcast:15, row_bcast:31
}

// One workgroup per (sequence, head). The threshold weight is found by its
// bytes, the highest first: a histogram in LDS of the candidates that match
// the bytes found so far, its running count from the top taken by every wave
// for itself, so that a byte costs one barrier. Weights have few first bytes
// (their signs and exponents), at which a wave's lanes would queue: that
// histogram is eight, a lane's by its number. Then, in one scan, the rows above
// the threshold and the first ones at it, in order.
//
// A thread has kPer rows side by side. Up to 16 * 1024 rows (CACHED) their keys
// stay in its registers over the five passes, 8 or 16 a thread; longer accounts
// are read again, stretch by stretch. What it waits for is latency: 8 x 8
// accounts of 8192 weights 13.5 us, 2 MB.
template <int kPer, bool CACHED>
__global__ __launch_bounds__(kSelectThreads) void mx4_select_kernel(SelectArgs a) {
    constexpr uint32_t kStretch = kPer * kSelectThreads;
    constexpr int kCopies = 8;
    __shared__ __attribute__((aligned(16))) uint32_t hist0[256][kCopies];
    __shared__ uint32_t hist[3][256];
    __shared__ uint32_t wave_above[kSelectThreads / 64], wave_equal[kSelectThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* w = a.weights + blockIdx.x * a.weight_stride;
    const uint32_t lo = a.first, hi = a.count - a.recent;  // the candidates
    uint32_t want = a.keep - a.first - a.recent;
    const bool any = want > 0, vec = (reinterpret_cast<uintptr_t>(w) & 15u) == 0;
    (&hist0[0][0])[tid] = (&hist0[0][0])[tid + kSelectThreads] = 0;
    if (tid < 3 * 256) (&hist[0][0])[tid] = 0;
    auto count = [&](int pass, uint32_t byte) { atomicAdd(pass == 0 ? &hist0[byte][lane % kCopies] : &hist[pass - 1][byte], 1u); };

    uint32_t key[kPer];
    float value[kPer];
    auto load = [&](uint32_t base) {
        const uint32_t j0 = base + tid * kPer;
        if (vec && j0 + kPer <= a.count) {
#pragma unroll
            for (int e = 0; e < kPer; e += 4) {
                const float4 x = *reinterpret_cast<const float4*>(w + j0 + e);
                value[e] = x.x;
                value[e + 1] = x.y;
                value[e + 2] = x.z;
                value[e + 3] = x.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < kPer; ++e) value[e] = j0 + e < a.count ? w[j0 + e] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < kPer; ++e) key[e] = weight_key(value[e]);
    };
    if (CACHED) load(0);
    uint32_t prefix = 0, mask = 0;
    __syncthreads();
    if (any) {
#pragma unroll
        for (int pass = 0; pass < 4; ++pass) {
            const int shift = 24 - 8 * pass;
            if constexpr (CACHED) {
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    const uint32_t j = tid * kPer + e;
                    if (j >= lo && j < hi && (key[e] & mask) == prefix) count(pass, key[e] >> shift & 255);
                }
            } else {
                // Counting asks for no order: lanes side by side.
                for (uint32_t base = lo; base < hi; base += kStretch) {
#pragma unroll
                    for (int e = 0; e < kPer; ++e) {
                        const uint32_t j = base + e * kSelectThreads + tid;
                        value[e] = j < hi ? w[j] : 0.0f;
                    }
#pragma unroll
                    for (int e = 0; e < kPer; ++e) {
                        const uint32_t k = weight_key(value[e]);
                        if (base + e * kSelectThreads + tid < hi && (k & mask) == prefix) count(pass, k >> shift & 255);
                    }
                }
            }
            __syncthreads();
            // Lane l has the bytes 252 - 4 l to 255 - 4 l; the byte sought is
            // the first from the top whose count reaches `want`.
            uint32_t bin[4], mine = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int byte = 255 - 4 * lane - x;
                if (pass == 0) {
                    const uint4* c = reinterpret_cast<const uint4*>(hist0[byte]);
                    bin[x] = c[0].x + c[0].y + c[0].z + c[0].w + c[1].x + c[1].y + c[1].z + c[1].w;
                } else {
                    bin[x] = hist[pass - 1][byte];
                }
                mine += bin[x];
            }
            const uint32_t upto = scan64(mine);
            const int at = __ffsll(static_cast<unsigned long long>(__ballot(upto >= want))) - 1;
            uint32_t left = want - (upto - mine), byte = 255 - 4 * lane;
#pragma unroll
            for (int x = 0; x < 3; ++x)
                if (byte == 255u - 4 * lane - x && bin[x] < left) {
                    left -= bin[x];
                    --byte;
                }
            want = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(left), at));
            prefix |= static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(byte), at)) << shift;
            mask |= 255u << shift;
        }
    }
    // Kept: the forced rows and those above the threshold, and the first
    // `want` of those at it (none where no candidate is wanted).
    uint32_t above_base = 0, equal_base = 0;
    for (uint32_t base = 0; base < a.count; base += kStretch) {
        if (!CACHED) load(base);
        uint32_t above = 0, equal = 0;  // a bit a row
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const uint32_t j = base + tid * kPer + e;
            const bool forced = j < lo || j >= hi;
            if (j < a.count) {
                if (forced || (any && key[e] > prefix)) above |= 1u << e;
                if (!forced && any && key[e] == prefix) equal |= 1u << e;
            }
        }
        const uint32_t own_a = static_cast<uint32_t>(__popc(above)), own_e = static_cast<uint32_t>(__popc(equal));
        uint32_t na = scan64(own_a), ne = scan64(own_e);
        if (lane == 63) {
            wave_above[wave] = na;
            wave_equal[wave] = ne;
        }
        __syncthreads();  // also: every read of this stretch of weights is done
        na += above_base - own_a;
        ne += equal_base - own_e;
#pragma unroll
        for (int i = 0; i < kSelectThreads / 64; ++i) {
            const uint32_t va = wave_above[i], ve = wave_equal[i];
            if (i < wave) {
                na += va;
                ne += ve;
            }
            above_base += va;
            equal_base += ve;
        }
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const bool is_above = above >> e & 1, is_equal = equal >> e & 1;
            if (is_above || (is_equal && ne < want)) {
                const uint32_t to = na + min(ne, want);
                a.indices[static_cast<uint64_t>(blockIdx.x) * a.keep + to] = base + tid * kPer + e;
                a.weights_out[blockIdx.x * a.out_stride + to] = value[e];
            }
            na += is_above;
            ne += is_equal;
        }
        if (!CACHED) __syncthreads();
    }
    // The rows that come next start at nothing.
    for (uint32_t j = a.keep + tid; j < a.out_rows; j += kSelectThreads) a.weights_out[blockIdx.x * a.out_stride + j] = 0.0f;
}

// The NB bytes of row r of a unit (`from`, as aligned as NB's power of two)
// into the unit's dwords.
template <int NB>
__device__ __forceinline__ void take_row(const uint8_t* from, int r, uint32_t (&code)[NB]) {
    if constexpr (NB % 4 == 0) {
#pragma unroll
        for (int w = 0; w < NB / 4; ++w) code[r * (NB / 4) + w] = reinterpret_cast<const uint32_t*>(from)[w];
    } else if constexpr (NB % 2 == 0) {
#pragma unroll
        for (int w = 0; w < NB / 2; ++w) {
            const int at = r * (NB / 2) + w;  // half dword of the unit
            code[at / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(from)[w]) << (16 * (at % 2));
        }
    } else {
#pragma unroll
        for (int p = 0; p < NB; ++p) {
            const int at = r * NB + p;
            code[at / 4] |= static_cast<uint32_t>(from[p]) << (8 * (at % 4));
        }
    }
}

// Rows of `src` to rows 0 .. keep - 1 of `dst`: row indices[i], or i itself
// where indices is null. 16 lanes a group of four rows, as for a write;
// blockIdx.y: the keys' or the values' store. A kept row is 4 NB bytes of each of
// its group's lines, so that the groups with a kept row are read whole: 2050 of
// 8192 rows of 64 heads of 128 in 19 us, about 44 MB of lines read and 18 written
// (23 us with a row's loads after the last one's). In place the rows go by way of
// the workspace, a second launch: they may move across workgroups.
struct MoveArgs {
    StoreArgs src[2], dst[2];
    const uint32_t* indices;
    uint32_t keep, groups_touched, units;
};
template <int NB>
__global__ __launch_bounds__(256) void mx4_move_kernel(MoveArgs a) {
    const uint32_t u = blockIdx.x * 16 + (threadIdx.x >> 4);
    const uint32_t n = threadIdx.x & 15;
    if (u >= a.units) return;
    const StoreArgs &src = a.src[blockIdx.y], &dst = a.dst[blockIdx.y];
    const uint32_t group = u % a.groups_touched, bh = u / a.groups_touched;
    const uint32_t h = bh % dst.heads, b = bh / dst.heads;
    const int hi = static_cast<int>(min(4u, a.keep - group * 4));
    uint32_t code[NB], row[4];
    uint32_t scale = 0;  // of block p = n
#pragma unroll
    for (int p = 0; p < NB; ++p) code[p] = 0;
    // A last group's rows past `keep` are read as its last one, and not written.
#pragma unroll
    for (int r = 0; r < 4; ++r) row[r] = group * 4 + min(r, hi - 1);
    if (a.indices)
#pragma unroll
        for (int r = 0; r < 4; ++r) row[r] = a.indices[static_cast<uint64_t>(bh) * a.keep + row[r]];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        take_row<NB>(unit_ptr<NB>(src, b, h, row[r] / 4, n) + (row[r] % 4) * NB, r, code);
        const uint32_t x = scale_ptr<NB>(src, b, h, row[r] / 4)[4 * min(n, NB - 1u) + row[r] % 4];
        scale |= x << (8 * r);
    }
    uint8_t* to = unit_ptr<NB>(dst, b, h, group, n);
    uint8_t* sto = scale_ptr<NB>(dst, b, h, group) + 4 * n;
    if (hi == 4) {
        __builtin_memcpy(__builtin_assume_aligned(to, NB % 4 == 0 ? 16 : NB % 2 == 0 ? 8 : 4), code, 4 * NB);
        if (n < NB) *reinterpret_cast<uint32_t*>(sto) = scale;
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (r >= hi) continue;
#pragma unroll
        for (int p = 0; p < NB; ++p) {
            const int at = r * NB + p;
            to[at] = static_cast<uint8_t>(code[at / 4] >> (8 * (at % 4)));
        }
        if (n < NB) sto[r] = static_cast<uint8_t>(scale >> (8 * r));
    }
}

mhip_status move_rows(mhip_ctx* ctx, MoveArgs& a, uint64_t batch, uint64_t heads, uint64_t nb) {
    a.groups_touched = static_cast<uint32_t>(mhip::ceil_div(a.keep, 4));
    const uint64_t units = batch * heads * a.groups_touched, blocks = mhip::ceil_div(units, 16);
    if (blocks >= (1ULL << 24)) return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "kv-evict: too many rows");
    a.units = static_cast<uint32_t>(units);
    const dim3 grid(static_cast<unsigned>(blocks), 2);
    switch (nb) {
        case 1: mhip::launch(ctx, mx4_move_kernel<1>, grid, dim3(256), 0, a); break;
        case 2: mhip::launch(ctx, mx4_move_kernel<2>, grid, dim3(256), 0, a); break;
        case 3: mhip::launch(ctx, mx4_move_kernel<3>, grid, dim3(256), 0, a); break;
        case 4: mhip::launch(ctx, mx4_move_kernel<4>, grid, dim3(256), 0, a); break;
        case 5: mhip::launch(ctx, mx4_move_kernel<5>, grid, dim3(256), 0, a); break;
        case 6: mhip::launch(ctx, mx4_move_kernel<6>, grid, dim3(256), 0, a); break;
        case 7: mhip::launch(ctx, mx4_move_kernel<7>, grid, dim3(256), 0, a); break;
        default: mhip::launch(ctx, mx4_move_kernel<8>, grid, dim3(256), 0, a); break;
    }
    return mhip::check_launch("kv-evict (move)");
}

mhip_status check_rows(const mhip_mx4_store* s, uint64_t count, uint64_t row_offset, const char* what) {
    mhip_status st = mhip::mx4_check(s, what);
    if (st != MHIP_OK) return st;
    if (row_offset > s->capacity || count > s->capacity - row_offset)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED,
                          std::string(what) + " of " + std::to_string(count) + " rows at " +
                              std::to_string(row_offset) + " exceeds the store's " + std::to_string(s->capacity) +
                              " rows");
    return MHIP_OK;
}

bool overlap(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + b_bytes && y < x + a_bytes;
}

uint64_t span(const mhip_mx4_store& s) {
    const uint64_t batch = s.batch ? s.batch : 1;
    const uint64_t stride = s.batch_stride ? s.batch_stride : mhip::mx4_bytes(s.capacity, s.kv_heads, s.head_dimension);
    return (batch - 1) * stride + mhip::mx4_used_bytes(s.capacity, s.kv_heads, s.head_dimension);
}

}  // namespace

extern "C" uint64_t mhip_kv_mx4_bytes(uint64_t capacity, uint64_t kv_heads, uint64_t head_dimension) {
    mhip_mx4_store s = {capacity, kv_heads, head_dimension, 1, 0};
    return mhip::mx4_check(&s, "kv store") == MHIP_OK ? mhip::mx4_bytes(capacity, kv_heads, head_dimension) : 0;
}

extern "C" mhip_status mhip_kv_write_mx4(mhip_ctx* ctx, void* store, const mhip_mx4_store* shape, const float* rows,
                                         uint64_t count, uint64_t row_offset) {
    MHIP_REQUIRE_CTX(ctx);
    mhip_status st = check_rows(shape, count, row_offset, "kv-write");
    if (st != MHIP_OK) return st;
    // A captured write may move down by up to the rows left after it; the
    // groups that it touches then depend on the offset, so one more is visited.
    const uint64_t* advance =
        mhip::advance_ptr(ctx, MHIP_ADVANCE_ROW_OFFSET, shape->capacity - (row_offset + count));
    if (count == 0) return MHIP_OK;
    if (!store || !rows) return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "kv-write: null buffer");
    if (!mhip::aligned16(store)) return mhip::fail(MHIP_LAYOUT_UNSUPPORTED, "kv-write: the store must be 16-byte aligned");
    const uint64_t batch = shape->batch ? shape->batch : 1, nb = mhip::mx4_blocks(shape->head_dimension);
    const uint64_t touched = advance ? mhip::ceil_div(count + 3, 4) : (row_offset + count - 1) / 4 - row_offset / 4 + 1;
    const uint64_t units = batch * touched * shape->kv_heads, blocks = mhip::ceil_div(units, 16);
    // A grid has fewer than 2^32 threads.
    if (blocks >= (1ULL << 24)) return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "kv-write: too many rows");
    const StoreArgs s = store_args(*shape, store);
    const dim3 grid(static_cast<unsigned>(blocks)), block(256);
    const uint32_t t = static_cast<uint32_t>(touched), n = static_cast<uint32_t>(units);
    switch (nb) {
        case 1: mhip::launch(ctx, mx4_write_kernel<1>, grid, block, 0, rows, s, count, row_offset, advance, t, n); break;
        case 2: mhip::launch(ctx, mx4_write_kernel<2>, grid, block, 0, rows, s, count, row_offset, advance, t, n); break;
        case 3: mhip::launch(ctx, mx4_write_kernel<3>, grid, block, 0, rows, s, count, row_offset, advance, t, n); break;
        case 4: mhip::launch(ctx, mx4_write_kernel<4>, grid, block, 0, rows, s, count, row_offset, advance, t, n); break;
        case 5: mhip::launch(ctx, mx4_write_kernel<5>, grid, block, 0, rows, s, count, row_offset, advance, t, n); break;
        case 6: mhip::launch(ctx, mx4_write_kernel<6>, grid, block, 0, rows, s, count, row_offset, advance, t, n); break;
        case 7: mhip::launch(ctx, mx4_write_kernel<7>, grid, block, 0, rows, s, count, row_offset, advance, t, n); break;
        default: mhip::launch(ctx, mx4_write_kernel<8>, grid, block, 0, rows, s, count, row_offset, advance, t, n); break;
    }
    return mhip::check_launch("kv-write (4-bit)");
}

extern "C" mhip_status mhip_kv_read_mx4(mhip_ctx* ctx, const void* store, const mhip_mx4_store* shape, float* rows,
                                        uint64_t count, uint64_t row_offset) {
    MHIP_REQUIRE_CTX(ctx);
    mhip_status st = check_rows(shape, count, row_offset, "kv-read");
    if (st != MHIP_OK || count == 0) return st;
    if (!store || !rows) return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "kv-read: null buffer");
    if (!mhip::aligned16(store)) return mhip::fail(MHIP_LAYOUT_UNSUPPORTED, "kv-read: the store must be 16-byte aligned");
    const uint64_t batch = shape->batch ? shape->batch : 1, nb = mhip::mx4_blocks(shape->head_dimension);
    const uint64_t touched = (row_offset + count - 1) / 4 - row_offset / 4 + 1;
    const uint64_t units = batch * touched * shape->kv_heads, blocks = mhip::ceil_div(units, 16);
    if (blocks >= (1ULL << 24)) return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "kv-read: too many rows");
    const StoreArgs s = store_args(*shape, store);
    const dim3 grid(static_cast<unsigned>(blocks)), block(256);
    const uint32_t t = static_cast<uint32_t>(touched), n = static_cast<uint32_t>(units);
    switch (nb) {
        case 1: mhip::launch(ctx, mx4_read_kernel<1>, grid, block, 0, rows, s, count, row_offset, t, n); break;
        case 2: mhip::launch(ctx, mx4_read_kernel<2>, grid, block, 0, rows, s, count, row_offset, t, n); break;
        case 3: mhip::launch(ctx, mx4_read_kernel<3>, grid, block, 0, rows, s, count, row_offset, t, n); break;
        case 4: mhip::launch(ctx, mx4_read_kernel<4>, grid, block, 0, rows, s, count, row_offset, t, n); break;
        case 5: mhip::launch(ctx, mx4_read_kernel<5>, grid, block, 0, rows, s, count, row_offset, t, n); break;
        case 6: mhip::launch(ctx, mx4_read_kernel<6>, grid, block, 0, rows, s, count, row_offset, t, n); break;
        case 7: mhip::launch(ctx, mx4_read_kernel<7>, grid, block, 0, rows, s, count, row_offset, t, n); break;
        default: mhip::launch(ctx, mx4_read_kernel<8>, grid, block, 0, rows, s, count, row_offset, t, n); break;
    }
    return mhip::check_launch("kv-read (4-bit)");
}

extern "C" mhip_status mhip_kv_evict_mx4(mhip_ctx* ctx, const void* k_store, const void* v_store, const float* weights,
                                         const mhip_mx4_store* shape, const mhip_kv_evict_params* p, void* k_out,
                                         void* v_out, const mhip_mx4_store* out_shape, float* weights_out,
                                         uint32_t* indices) {
    MHIP_REQUIRE_CTX(ctx);
    mhip_status st = mhip::mx4_check(shape, "kv-evict");
    if (st == MHIP_OK) st = mhip::mx4_check(out_shape, "kv-evict");
    if (st != MHIP_OK) return st;
    if (!p) return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "kv-evict: null params");
    const uint64_t batch = shape->batch ? shape->batch : 1;
    const uint64_t heads = shape->kv_heads, d = shape->head_dimension;
    if (out_shape->kv_heads != heads || out_shape->head_dimension != d ||
        (out_shape->batch ? out_shape->batch : 1) != batch)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "kv-evict: the stores differ in heads, head dimension or batch");
    if (p->key_count > shape->capacity)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "kv-evict: key_count " + std::to_string(p->key_count) +
                                                      " exceeds the store's " + std::to_string(shape->capacity) + " rows");
    if (p->keep > p->key_count)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "kv-evict: cannot keep " + std::to_string(p->keep) + " of " +
                                                      std::to_string(p->key_count) + " rows");
    if (p->keep > out_shape->capacity)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "kv-evict: " + std::to_string(p->keep) +
                                                      " rows exceed the output store's " +
                                                      std::to_string(out_shape->capacity));
    if (p->first > p->keep || p->recent > p->keep - p->first)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "kv-evict: the first and recent rows exceed the rows to keep");
    const uint64_t w_stride = p->weight_stride ? p->weight_stride : shape->capacity;
    const uint64_t o_stride = p->weight_out_stride ? p->weight_out_stride : out_shape->capacity;
    if (w_stride < p->key_count || o_stride < out_shape->capacity)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "kv-evict: the weights' stride is below their row count");
    // The rows that stay depend on a key count that no replay offset moves.
    (void)mhip::advance_ptr(ctx, MHIP_ADVANCE_KEY_COUNT, 0);
    if (out_shape->capacity == 0) return MHIP_OK;
    if (!k_store || !v_store || !weights || !k_out || !v_out || !weights_out)
        return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "kv-evict: null buffer");
    if (!mhip::aligned16(k_store) || !mhip::aligned16(v_store) || !mhip::aligned16(k_out) || !mhip::aligned16(v_out))
        return mhip::fail(MHIP_LAYOUT_UNSUPPORTED, "kv-evict: the stores must be 16-byte aligned");
    const uint64_t in_span = span(*shape), out_span = span(*out_shape);
    const bool same_shape = out_shape->capacity == shape->capacity &&
                            store_args(*out_shape, k_out).stride == store_args(*shape, k_store).stride;
    const bool in_place = k_out == k_store && v_out == v_store && same_shape;
    if (overlap(k_out, out_span, v_out, out_span) ||
        (!in_place && (overlap(k_store, in_span, k_out, out_span) || overlap(v_store, in_span, v_out, out_span) ||
                       overlap(k_store, in_span, v_out, out_span) || overlap(v_store, in_span, k_out, out_span))))
        return mhip::fail(MHIP_LAYOUT_UNSUPPORTED,
                          "kv-evict: the output stores overlap the stores (in place: the same stores and shape)");
    const uint64_t rows = batch * heads;
    if (rows >= (1ULL << 22)) return mhip::fail(MHIP_SHAPE_UNSUPPORTED, "kv-evict: too many heads");
    const uint64_t w_bytes = (rows - 1) * w_stride * 4 + p->key_count * 4;
    const uint64_t o_bytes = (rows - 1) * o_stride * 4 + out_shape->capacity * 4;
    if (!(weights_out == weights && w_stride == o_stride) && overlap(weights, w_bytes, weights_out, o_bytes))
        return mhip::fail(MHIP_LAYOUT_UNSUPPORTED, "kv-evict: the weights overlap (in place: the same buffer and stride)");

    // Scratch: the indices, unless the caller takes them, and for an eviction
    // in place the kept rows of both stores before they are put back.
    const uint64_t index_bytes = indices ? 0 : (rows * p->keep * 4 + 255) / 256 * 256;
    const uint64_t one = mhip::mx4_bytes(p->keep, heads, d);
    const uint64_t bytes = index_bytes + (in_place ? 2 * batch * one : 0);
    uint8_t* scratch = nullptr;
    const mhip::CaptureGrowth growth(ctx, true);
    if (bytes) {
        void* ws = nullptr;
        st = mhip::workspace(ctx, bytes, &ws);
        if (st != MHIP_OK) return st;
        scratch = static_cast<uint8_t*>(ws);
    }
    SelectArgs sel;
    sel.weights = weights;
    sel.weights_out = weights_out;
    sel.indices = indices ? indices : reinterpret_cast<uint32_t*>(scratch);
    sel.weight_stride = w_stride;
    sel.out_stride = o_stride;
    sel.count = static_cast<uint32_t>(p->key_count);
    sel.keep = static_cast<uint32_t>(p->keep);
    sel.first = static_cast<uint32_t>(p->first);
    sel.recent = static_cast<uint32_t>(p->recent);
    sel.out_rows = static_cast<uint32_t>(out_shape->capacity);
    const dim3 grid(static_cast<unsigned>(rows)), block(kSelectThreads);
    if (p->key_count <= kSelectThreads * 8)
        mhip::launch(ctx, mx4_select_kernel<8, true>, grid, block, 0, sel);
    else if (p->key_count <= kSelectThreads * 16)
        mhip::launch(ctx, mx4_select_kernel<16, true>, grid, block, 0, sel);
    else
        mhip::launch(ctx, mx4_select_kernel<16, false>, grid, block, 0, sel);
    st = mhip::check_launch("kv-evict (select)");
    if (st != MHIP_OK || p->keep == 0) return st;

    const uint64_t nb = mhip::mx4_blocks(d);
    MoveArgs mv;
    mv.indices = sel.indices;
    mv.keep = sel.keep;
    mv.src[0] = store_args(*shape, k_store);
    mv.src[1] = store_args(*shape, v_store);
    mv.dst[0] = store_args(*out_shape, k_out);
    mv.dst[1] = store_args(*out_shape, v_out);
    if (!in_place) return move_rows(ctx, mv, batch, heads, nb);
    const mhip_mx4_store held = {p->keep, heads, d, batch, 0};
    MoveArgs back = mv;
    mv.dst[0] = store_args(held, scratch + index_bytes);
    mv.dst[1] = store_args(held, scratch + index_bytes + batch * one);
    st = move_rows(ctx, mv, batch, heads, nb);
    if (st != MHIP_OK) return st;
    back.src[0] = mv.dst[0];
    back.src[1] = mv.dst[1];
    back.indices = nullptr;
    return move_rows(ctx, back, batch, heads, nb);
}
