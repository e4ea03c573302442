// gsd_attention_bwd.hip — cross attention, backward:
//   delta = sum_d do o                    (a row's sum of p dp)
//   p = 2^(s log2e - lse),  dp = do v^T,  ds = p (dp - delta)
//   dv = p^T do,  dk = scale ds^T q,  dq = scale ds k
// with p formed again from q, k and the forward's lse.
//
// Three kernels.  delta reads do and o once.  dk and dv: a wave holds 32 keys
// (k, v and both sums in registers) and walks the rows; s = Q K^T and dp = dO
// V^T leave a key's column in a lane, so p and ds are operand B of dv^T = dO^T p
// and dk^T = Q^T ds.  dq: a wave holds 32 rows and walks the keys; s^T, dp^T,
// then dq^T = K^T ds^T.  s and dp are formed in both, seven products where five
// would do: one kernel for all three gradients would have to add dq over the key
// blocks with atomics, whose order changes results, or through memory.
//
// As in the forward, matrix products and vector instructions bound them.  4096 x
// 32400, 16 heads of 128 in groups of 4: dk and dv 2.00 to 2.09 ms by card (1.04 to
// 1.09 PFLOP/s; 0.52 of a SIMD's cycles with a matrix instruction, 0.35 with a vector
// one, 0.08 with both), dq 1.30 to 1.38 ms (1.18 to 1.25; 0.65, 0.33 and 0.10), delta 11
// us (5 TB/s).
#include "gsd_attention.h"

namespace gsd {

AttnArgs attention_args(const gsd_attention& g, int32_t* list);
hipError_t launch_key_list(const AttnArgs& a, hipStream_t st);
int64_t split_parts(int64_t blocks, int64_t tiles, int64_t least, int64_t per_unit);

namespace {

constexpr int kHeld = 128;  // rows (dq) or keys (dk, dv) that a work-group holds
constexpr int kDeltaRows = 64;

// Few terms (kFewTerms) that the sizes show make for kernels of their own (kFew): making up
// for the roundings makes dk and dv of 64 x 32400, 16 heads of 128, 7% and dq 10% longer
// (199 and 62 us) and 4096 x 64 no longer (21 and 14 us).  Where only a batch's length or
// mask shows them, the kernels' work-groups see it and take that path.
bool few_terms(int64_t rows, int64_t keys) { return rows <= kFewTerms || keys <= kFewTerms; }

struct GradArgs {
    AttnArgs f;
    const char* d_o;
    int64_t dob, dol, doh;  // bytes
    // [batch kv_heads, 2, rows]: shift - lse (-infinity for a row without a key), -delta
    float* stat;
    // fp16: [batch kv_heads, 2, top_blocks], max |do| (a row's norm) and max |delta| per
    // block of rows, and [batch kv_heads, value_blocks], max |v| per block of keys
    float *top, *value_top;
    int32_t top_blocks, value_blocks;
    char *dq, *dk, *dv;
    float *partial_dq, *partial_dk, *partial_dv;
};

struct RowAt {
    int64_t l;
    int head;
};
__device__ __forceinline__ RowAt row_at(const AttnArgs& a, int kvh, int row) {
    const uint32_t l = (uint32_t)row / (uint32_t)a.group;
    return RowAt{l, kvh * a.group + row - (int)l * a.group};
}

// Whether a batch's key takes part.
__device__ __forceinline__ bool key_valid(const AttnArgs& a, int64_t b, int64_t key) {
    if (key >= admitted_keys(a, (int)b)) return false;
    return !a.mask || a.mask[b * a.mb + key * a.ms] != 0;
}

// dk and dv of keys that take no part: a thread per eight values of both.
__device__ __forceinline__ void zero_keys(const GradArgs& g, uint32_t group) {
    const AttnArgs& a = g.f;
    const int units = a.kv_heads * a.dim / 8;
    const int64_t id = (int64_t)group * kThreads + threadIdx.x;
    const int64_t row = id / units;
    if (row >= (int64_t)a.batch * a.keys) return;
    const int64_t b = row / a.keys;
    if (key_valid(a, b, row - b * a.keys)) return;
    store_any(g.dk + 16 * id, u32x4{0, 0, 0, 0});
    store_any(g.dv + 16 * id, u32x4{0, 0, 0, 0});
}

// The maximum over a work-group.
__device__ __forceinline__ float group_max(float v, float (&part)[kWaves]) {
    v = wave_max(v);
    if (lane_id() == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    return fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
}

// max |v| over 64 keys that take part, 16 lanes per key.
template <typename T>
__device__ __forceinline__ void value_norms(const GradArgs& g, uint32_t group,
                                            float (&part)[kWaves]) {
    const AttnArgs& a = g.f;
    const int bh = (int)(group / g.value_blocks), block = (int)(group % g.value_blocks);
    const int b = bh / a.kv_heads, kvh = bh % a.kv_heads;
    const int c = threadIdx.x % 16;
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < kDeltaRows / 16; ++j) {
        const int64_t key = (int64_t)block * kDeltaRows + j * 16 + (int)threadIdx.x / 16;
        float square = 0.0f;
        if (8 * c < a.dim && key_valid(a, b, key)) {
            const auto x = load_any<typename T::vec8>(a.v + b * a.vb + key * a.vs + kvh * a.vh + 16 * c);
#pragma unroll
            for (int i = 0; i < 8; ++i) square = __builtin_fmaf((float)x[i], (float)x[i], square);
        }
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) square += __shfl_xor(square, d);
        top = fmaxf(top, square);
    }
    top = group_max(top, part);
    if (threadIdx.x == 0) g.value_top[group] = sqrtf(top);
}

// ---- delta: 16 lanes per row of up to 128 elements ----
// The work-groups behind those of the rows find the largest |v| (fp16) and write the
// zeros of keys that take no part: 2 x 1237 x 8260, 8 heads of 128, takes 390 us with
// lengths, forward and backward, 396 with a launch for the zeros, and 2 x 32 x 300, which
// the host bounds, 86 and 89.
template <typename T>
__global__ __launch_bounds__(kThreads) void delta_kernel(GradArgs g) {
    const AttnArgs& a = g.f;
    __shared__ float s_top[kWaves], s_delta[kWaves];
    const uint32_t heads = (uint32_t)a.batch * a.kv_heads;
    uint32_t groups = heads * g.top_blocks;
    if (blockIdx.x >= groups) {
        const uint32_t values = T::kScaled ? heads * g.value_blocks : 0;
        if (blockIdx.x - groups < values)
            value_norms<T>(g, blockIdx.x - groups, s_top);
        else
            zero_keys(g, blockIdx.x - groups - values);
        return;
    }
    const int bh = (int)(blockIdx.x / g.top_blocks);
    const int block = (int)(blockIdx.x % g.top_blocks);
    const int b = bh / a.kv_heads, kvh = bh % a.kv_heads;
    const int c = threadIdx.x % 16;
    const int64_t queries = a.rows / a.group;
    float top = 0.0f, top_delta = 0.0f;
#pragma unroll
    for (int j = 0; j < kDeltaRows / 16; ++j) {
        const int row = block * kDeltaRows + j * 16 + (int)threadIdx.x / 16;
        float dot = 0.0f, square = 0.0f;
        if (row < a.rows && 8 * c < a.dim) {
            const RowAt at = row_at(a, kvh, row);
            const auto x = load_any<typename T::vec8>(g.d_o + b * g.dob + at.l * g.dol +
                                                      at.head * g.doh + 16 * c);
            const int64_t from = ((b * queries + at.l) * a.heads + at.head) * (int64_t)a.dim + 8 * c;
            const auto y = load_any<typename T::vec8>(a.o + 2 * from);
            typename T::vec8 z;
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = (typename T::elem)0.0f;
            if (a.o_low) z = load_any<typename T::vec8>(a.o_low + 2 * from);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                dot = __builtin_fmaf((float)x[i], (float)y[i] + (float)z[i], dot);
                if (T::kScaled) square = __builtin_fmaf((float)x[i], (float)x[i], square);
            }
        }
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) {
            dot += __shfl_xor(dot, d);
            if (T::kScaled) square += __shfl_xor(square, d);
        }
        if (c == 0 && row < a.rows) {
            const float lse = a.lse[(int64_t)bh * a.rows + row];
            float* const to = g.stat + 2 * (int64_t)bh * a.rows + row;
            to[0] = lse == -__builtin_inff() ? lse : T::kGradShift - lse;
            to[a.rows] = -dot;
        }
        top = fmaxf(top, square);
        top_delta = fmaxf(top_delta, fabsf(dot));
    }
    if (!T::kScaled) return;
    top = group_max(top, s_top);
    top_delta = group_max(top_delta, s_delta);
    if (threadIdx.x == 0) {
        float* const to = g.top + 2 * (int64_t)bh * g.top_blocks + block;
        to[0] = sqrtf(top);
        to[g.top_blocks] = top_delta;
    }
}

// The largest of n, by a wave.
__device__ __forceinline__ float largest(const float* v, int n) {
    float top = 0.0f;
    for (int i = lane_id(); i < n; i += kWave) top = fmaxf(top, v[i]);
    return wave_max(top);
}

// The power of two that ds is scaled by before it is rounded, from a bound on |dp -
// delta|: |do| |v| + |delta|, of a row for dq and of a key for dk, which take it out of
// their sums again.  It brings the bound to [2^14, 2^15), so that ds, p times that with p
// at most 1, neither overflows fp16 nor loses digits before it is 2^-28 of the bound (p of
// 1 / 32400 and a bound that is 2^5 too high leave 2^8).  1 where the bound is 0 or not
// finite.  In what follows a lane holds half of the row's or key's elements in `held`.
template <typename T, int N>
__device__ __forceinline__ float held_norm(const typename T::vec8 (&held)[N]) {
    float square = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            square = __builtin_fmaf((float)held[j][i], (float)held[j][i], square);
    return sqrtf(square + other_half(square));
}
__device__ __forceinline__ float scale_of(float bound) {
    if (!(bound > 0.0f) || !(bound < __builtin_inff())) return 1.0f;
    return __builtin_ldexpf(1.0f, 15 - __builtin_amdgcn_frexp_expf(bound));
}
template <typename T, int N>
__device__ __forceinline__ float row_scale(const GradArgs& g, int bh,
                                           const typename T::vec8 (&d_o)[N], float delta) {
    if (!T::kScaled) return 1.0f;
    const float value = largest(g.value_top + (int64_t)bh * g.value_blocks, g.value_blocks);
    return scale_of(__builtin_fmaf(held_norm<T>(d_o), value, fabsf(delta)));
}
template <typename T, int N>
__device__ __forceinline__ float key_scale(const GradArgs& g, int bh,
                                           const typename T::vec8 (&v)[N]) {
    if (!T::kScaled) return 1.0f;
    const float* from = g.top + 2 * (int64_t)bh * g.top_blocks;
    const float d_o = largest(from, g.top_blocks), delta = largest(from + g.top_blocks, g.top_blocks);
    return scale_of(__builtin_fmaf(d_o, held_norm<T>(v), delta));
}

// Tiles of kRows of the problem's rows straight to LDS, one after the other, for q
// and do alike: row r lies at query r / G and the group's head r % G.  Where G
// divides kRows a lane's offset from its tile's first query is the same for every
// tile.
template <int DT, int kRows>
struct RowDma {
    using Tile = TileDma<DT, kRows>;
    static constexpr int kChunks = Tile::kChunks;
    const char* base;  // of the tile's first query
    uint32_t offset[kChunks];
    uint32_t ls, hs;  // strides, bytes: 65 ls + G hs < 2^31
    int group, dim, first;  // first: the head that the tile starts with

    __device__ __forceinline__ void place() {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            int r, c;
            Tile::place(threadIdx.x, i, r, c);
            const uint32_t at = (uint32_t)(r + first), l = at / (uint32_t)group;
            offset[i] = 8 * c < dim ? l * ls + (at - l * group) * hs + 16 * c : kOutside;
        }
    }
    // from: of the batch and the group's first head
    __device__ __forceinline__ void init(const char* from, int64_t l_stride, int64_t h_stride,
                                         int g, int d, int tile) {
        ls = (uint32_t)l_stride;
        hs = (uint32_t)h_stride;
        group = g;
        dim = d;
        const uint32_t row0 = (uint32_t)tile * kRows, l = row0 / (uint32_t)g;
        first = (int)(row0 - l * g);
        base = from + l * l_stride;
        place();
    }
    // left: rows of the problem from the tile's first on
    __device__ __forceinline__ void issue(int left, char* tile) const {
        const u32x4 from = buffer_at(base);
        const uint32_t to = lds_address(tile) + wave_id() * kChunks * 1024;
        if (left >= kRows) {
            dma16(from, offset, to);
        } else {
            const int thread = opaque(threadIdx.x);
            uint32_t some[kChunks];
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                int r, c;
                Tile::place(thread, i, r, c);
                some[i] = r < left ? offset[i] : kOutside;
            }
            dma16(from, some, to);
        }
    }
    __device__ __forceinline__ void next() {
        const int step = kRows / group, rest = kRows % group;
        base += (int64_t)step * ls;
        if (rest == 0) return;
        first += rest;
        if (first >= group) {
            first -= group;
            base += ls;
        }
        place();
    }
};

// Operand B held in registers: column l of 32, element 16 ks + 8 half ...
template <typename T, int DT>
__device__ __forceinline__ void hold(typename T::vec8 (&v)[DT / 16], const char* from, bool ok,
                                     int dim) {
    const int half = lane_id() >> 5;
#pragma unroll
    for (int ks = 0; ks < DT / 16; ++ks) {
        const int d = 16 * ks + 8 * half;
        u32x4 in{0, 0, 0, 0};
        if (ok && d < dim) in = load_any<u32x4>(from + 2 * d);
        v[ks] = __builtin_bit_cast(typename T::vec8, in);
    }
}

template <int N>
__device__ __forceinline__ void clear(f32x16 (&v)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) v[j][i] = 0.0f;
}

// A sum's column (element d = 32 db + 8 k + 4 half + i), times f, to memory.
template <typename T, int DT, bool kPartial>
__device__ __forceinline__ void put(const f32x16 (&v)[DT / 32], float f, void* to, int dim) {
    const int half = lane_id() >> 5;
#pragma unroll
    for (int db = 0; db < DT / 32; ++db)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int d = 32 * db + 8 * k + 4 * half;
            if (d >= dim) continue;
            if (kPartial) {
                f32x4 out;
#pragma unroll
                for (int i = 0; i < 4; ++i) out[i] = v[db][4 * k + i] * f;
                store_any(static_cast<float*>(to) + d, out);
            } else {
                typedef typename T::elem vec4 __attribute__((ext_vector_type(4)));
                vec4 out;
#pragma unroll
                for (int i = 0; i < 4; ++i) out[i] = (typename T::elem)(v[db][4 * k + i] * f);
                store_any(static_cast<char*>(to) + 2 * d, out);
            }
        }
}

template <typename T, int DT, int DC, bool kList, bool kFew>
__global__ __launch_bounds__(kThreads, 2) void dq_kernel(GradArgs g) {
    const AttnArgs& a = g.f;
    constexpr int kBytes = kTile * DT * 2;
    __shared__ __attribute__((aligned(256))) char s_k0[kBytes], s_v0[kBytes];
    __shared__ __attribute__((aligned(256))) char s_k1[kBytes], s_v1[kBytes];
    typedef typename T::vec8 vec8;

    const uint32_t id = work_of(blockIdx.x, a.blocks * a.parts * a.kv_heads);
    const uint32_t block = id % a.blocks;
    const uint32_t part = id / a.blocks % a.parts;
    const int bh = (int)(id / a.blocks / a.parts);
    const int b = bh / a.kv_heads, kvh = bh % a.kv_heads;
    const int lane = lane_id(), wave = wave_id();

    KeyDma<kList, DT> keys;
    keys.init(a, b, kvh);
    KeyWalk<kList> walk;
    walk.start(a, b, part);
    if (walk.more()) {
        walk.look_ahead();
        keys.fetch(walk, s_k0, s_v0);
    }

    const int row = (int)block * kHeld + wave * 32 + (lane & 31);
    const bool live = row < a.rows;
    const bool busy = (int)block * kHeld + wave * 32 < a.rows;  // else it only loads and waits
    const RowAt at = row_at(a, kvh, live ? row : 0);
    vec8 q[DC / 16], d_o[DC / 16];
    hold<T, DC>(q, a.q + b * a.qb + at.l * a.ql + at.head * a.qh, live, a.dim);
    hold<T, DC>(d_o, g.d_o + b * g.dob + at.l * g.dol + at.head * g.doh, live, a.dim);
    float off = -__builtin_inff(), minus_delta = 0.0f;
    if (live) {
        const float* from = g.stat + 2 * (int64_t)bh * a.rows + row;
        off = from[0];
        minus_delta = from[a.rows];
    }
    // with the 2^kGradShift that p carries taken out
    const float ds_scale =
        row_scale<T>(g, bh, d_o, minus_delta) * __builtin_ldexpf(1.0f, -(int)T::kGradShift);
    f32x16 begin;  // dp's sums begin at -delta, which saves its addition to each
#pragma unroll
    for (int i = 0; i < 16; ++i) begin[i] = minus_delta;
    f32x16 dq[DC / 32];
    clear(dq);

    auto step = [&](auto low, const char* tile_k, const char* tile_v, char* next_k,
                    char* next_v) GSD_INLINE -> bool {
        constexpr bool kLow = decltype(low)::value;
        const int left = walk.left();
        walk.next();
        const bool more = walk.more();
        if (more) {
            walk.look_ahead();
            keys.fetch(walk, next_k, next_v);
        }
        if (busy)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
            f32x16 s, dp;
            // ahead of the other wave of the SIMD: where both have products to
            // issue they would reach their exponentials together
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.0f;
            dp = begin;
#pragma unroll
            for (int ks = 0; ks < DC / 16; ++ks) {
                s = T::mma(read_rows<T, DT>(tile_k, 32 * h, ks), q[ks], s);
                dp = T::mma(read_rows<T, DT>(tile_v, 32 * h, ks), d_o[ks], dp);
            }
            pace<DC / 16, 2, 2, 2>();
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale_log2, off));
                s[i] = p * (dp[i] * ds_scale);
                if constexpr (kLow) s[i] = formed(s[i]);
            }
            if (left < kTile) {
                const int me = opaque(lane);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (past(h, i, me, left)) s[i] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const vec8 ds = pack<T>(s, k);
#pragma unroll
                for (int db = 0; db < DC / 32; ++db) {
                    const vec8 kt = read_columns<T, DT>(tile_k, 32 * h + 16 * k, db);
                    dq[db] = T::mma(kt, ds, dq[db]);
                    if constexpr (kLow) dq[db] = T::mma(kt, pack_low<T>(s, k), dq[db]);
                }
            }
            if constexpr (!kLow) pace<DC / 16, 2, 1, 2>();
            __builtin_amdgcn_sched_barrier(0);
        }
        if (more) {
            dma_wait();
            __syncthreads();
        }
        return more;
    };
    if (walk.more()) {
        dma_wait();
        __syncthreads();
        using Low = std::integral_constant<bool, kFew>;
        if (!kFew && __builtin_expect(walk.n <= kFewTerms, 0))
            step(std::true_type{}, s_k0, s_v0, s_k1, s_v1);
        else
            while (step(Low{}, s_k0, s_v0, s_k1, s_v1) && step(Low{}, s_k1, s_v1, s_k0, s_v0)) {
            }
    }
    if (!live) return;
    const float f = a.scale / (ds_scale * __builtin_ldexpf(1.0f, (int)T::kGradShift));
    if (a.parts == 1) {
        const int64_t queries = a.rows / a.group;
        put<T, DC, false>(dq, f, g.dq + 2 * (((b * queries + at.l) * a.heads + at.head) * (int64_t)a.dim),
                          a.dim);
    } else {
        const int64_t to = ((int64_t)part * a.batch * a.kv_heads + bh) * a.rows + row;
        put<T, DC, true>(dq, f, g.partial_dq + to * a.dim, a.dim);
    }
}

constexpr int kGradRows = 64;  // rows per tile

template <typename T, int DT, bool kFew>
__global__ __launch_bounds__(kThreads, kFew ? 2 : 3) void dkdv_kernel(GradArgs g) {
    const AttnArgs& a = g.f;
    constexpr int kRows = kGradRows;
    constexpr int kBytes = kRows * DT * 2;
    __shared__ __attribute__((aligned(256))) char s_q0[kBytes], s_g0[kBytes];
    __shared__ __attribute__((aligned(256))) char s_q1[kBytes], s_g1[kBytes];
    __shared__ __attribute__((aligned(256))) float s_stat0[2 * kRows], s_stat1[2 * kRows];
    typedef typename T::vec8 vec8;

    const uint32_t id = work_of(blockIdx.x, a.blocks * a.parts * a.kv_heads);
    const uint32_t block = id % a.blocks;
    const uint32_t part = id / a.blocks % a.parts;
    const int bh = (int)(id / a.blocks / a.parts);
    const int b = bh / a.kv_heads, kvh = bh % a.kv_heads;
    const int lane = lane_id(), wave = wave_id(), half = lane >> 5;

    // with a mask, the block's keys are the next of the list
    const int at_key = (int)block * kHeld + wave * 32 + (lane & 31);
    const int keys = a.list ? a.counts[b] : admitted_keys(a, b);
    const bool valid = at_key < keys;
    const bool busy = ballot(valid) != 0;  // else a wave only loads and waits
    const int64_t key = a.list && valid ? a.list[(int64_t)b * a.keys + at_key] : at_key;
    f32x16 dk[DT / 32], dv[DT / 32];
    clear(dk);
    clear(dv);
    float ds_scale = 1.0f;
    int t = (int)part * a.tiles_per_part, end = t + a.tiles_per_part;
    end = end < a.tiles ? end : a.tiles;

    // a work-group without a valid key has nothing to add
    if (__syncthreads_or(valid) && t < end) {
        const char* qbase = a.q + b * a.qb + (int64_t)kvh * a.group * a.qh;
        const char* gbase = g.d_o + b * g.dob + (int64_t)kvh * a.group * g.doh;
        // a wave each for the rows' two
        const char* stat_base =
            reinterpret_cast<const char*>(g.stat + (2 * (int64_t)bh + (wave & 1)) * a.rows);
        RowDma<DT, kRows> rq, rg;
        rq.init(qbase, a.ql, a.qh, a.group, a.dim, t);
        rg.init(gbase, g.dol, g.doh, a.group, a.dim, t);
        auto fetch = [&](char* to_q, char* to_g, float* to_stat) {
            const int left = a.rows - t * kRows;
            rq.issue(left, to_q);
            rg.issue(left, to_g);
            // a row past the end has q = do = 0, where any finite off leaves
            // nothing
            static_assert(kRows == kWave, "one load of a wave");
            if (wave < 2)
                dma4(buffer_at(stat_base + (int64_t)4 * kRows * t), lane < left ? 4 * lane : kOutside,
                     lds_address(to_stat + wave * kRows));
        };
        fetch(s_q0, s_g0, s_stat0);
        vec8 k[DT / 16], v[DT / 16];
        hold<T, DT>(k, a.k + b * a.kb + key * a.ks + kvh * a.kh, valid, a.dim);
        hold<T, DT>(v, a.v + b * a.vb + key * a.vs + kvh * a.vh, valid, a.dim);
        // with the 2^kGradShift that p carries taken out
        ds_scale = key_scale<T>(g, bh, v) * __builtin_ldexpf(1.0f, -(int)T::kGradShift);
        dma_wait();
        __syncthreads();
        auto step = [&](auto low, const char* tile_q, const char* tile_g, const float* stat,
                        char* next_q, char* next_g, float* next_stat) GSD_INLINE -> bool {
            constexpr bool kLow = decltype(low)::value;
            const bool more = ++t < end;
            if (more) {
                rq.next();
                rg.next();
                fetch(next_q, next_g, next_stat);
            }
            if (busy) {
                f32x16 s[2], dp[2];
                auto scores = [&](int h) {
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4) {
                        // dp's sums begin at -delta, which saves its addition to each
                        const f32x4 nd = *reinterpret_cast<const f32x4*>(
                            stat + kRows + 32 * h + 8 * i4 + 4 * half);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            s[h][4 * i4 + i] = 0.0f;
                            dp[h][4 * i4 + i] = nd[i];
                        }
                    }
#pragma unroll
                    for (int ks = 0; ks < DT / 16; ++ks) {
                        s[h] = T::mma(read_rows<T, DT>(tile_q, 32 * h, ks), k[ks], s[h]);
                        dp[h] = T::mma(read_rows<T, DT>(tile_g, 32 * h, ks), v[ks], dp[h]);
                    }
                };
                auto softmax = [&](int h) {
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4) {
                        const f32x4 of =
                            *reinterpret_cast<const f32x4*>(stat + 32 * h + 8 * i4 + 4 * half);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int j = 4 * i4 + i;
                            s[h][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][j], a.scale_log2, of[i]));
                            dp[h][j] = s[h][j] * (dp[h][j] * ds_scale);
                            if constexpr (kLow) dp[h][j] = formed(dp[h][j]);
                        }
                    }
                };
                auto sums = [&](int h) {
#pragma unroll
                    for (int b2 = 0; b2 < 2; ++b2) {
                        const vec8 p = pack<T>(s[h], b2), ds = pack<T>(dp[h], b2);
#pragma unroll
                        for (int db = 0; db < DT / 32; ++db) {
                            const vec8 gt = read_columns<T, DT>(tile_g, 32 * h + 16 * b2, db);
                            const vec8 qt = read_columns<T, DT>(tile_q, 32 * h + 16 * b2, db);
                            dv[db] = T::mma(gt, p, dv[db]);
                            dk[db] = T::mma(qt, ds, dk[db]);
                            if constexpr (kLow) {
                                dv[db] = T::mma(gt, pack_low<T>(s[h], b2), dv[db]);
                                dk[db] = T::mma(qt, pack_low<T>(dp[h], b2), dk[db]);
                            }
                        }
                    }
                };
                constexpr int kSteps = DT / 16;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    scores(h);
                    softmax(h);
                    sums(h);
                    if constexpr (!kLow) {
                        pace<kSteps, 2, 2, 3>();
                        pace<kSteps, 4, 2, 2>();
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (more) {
                dma_wait();
                __syncthreads();
            }
            return more;
        };
        auto all = [&](auto low) GSD_INLINE {
            while (step(low, s_q0, s_g0, s_stat0, s_q1, s_g1, s_stat1) &&
                   step(low, s_q1, s_g1, s_stat1, s_q0, s_g0, s_stat0)) {
            }
        };
        if (!kFew && __builtin_expect(keys <= kFewTerms, 0))
            all(std::true_type{});
        else
            all(std::integral_constant<bool, kFew>{});
    }
    if (!valid) return;  // their gradients are written as 0 with delta
    const float fk = a.scale / (ds_scale * __builtin_ldexpf(1.0f, (int)T::kGradShift));
    const float fv = __builtin_ldexpf(1.0f, -(int)T::kGradShift);
    if (a.parts == 1) {
        const int64_t to = 2 * (((b * a.keys + key) * a.kv_heads + kvh) * (int64_t)a.dim);
        put<T, DT, false>(dk, fk, g.dk + to, a.dim);
        put<T, DT, false>(dv, fv, g.dv + to, a.dim);
    } else {
        const int64_t to = (((int64_t)part * a.batch * a.kv_heads + bh) * a.keys + key) * a.dim;
        put<T, DT, true>(dk, fk, g.partial_dk + to, a.dim);
        put<T, DT, true>(dv, fv, g.partial_dv + to, a.dim);
    }
}

// The same for heads of 128, whose sums, k and v leave no room for a second wave
// on a SIMD, and one wave alone waits between its products and its exponentials.
// Two waves share 32 keys instead: each forms p and ds of one half of a tile's
// rows, one then adds dv, the other dk over all of them, and each passes the other
// what it does not add itself through LDS (packed as operands, 2 KB).  4096 x
// 32400, 16 heads of 128: 3.0 ms as above (and 512 registers), 2.0 ms so.
constexpr int kPairHeld = 64;

template <typename T, int DC, bool kFew>
__global__ __launch_bounds__(kThreads, 2) void dkdv_pair_kernel(GradArgs g) {
    const AttnArgs& a = g.f;
    constexpr int DT = 128, kRows = kGradRows;
    constexpr int kBytes = kRows * DT * 2;
    __shared__ __attribute__((aligned(256))) char s_q0[kBytes], s_g0[kBytes];
    __shared__ __attribute__((aligned(256))) char s_q1[kBytes], s_g1[kBytes];
    __shared__ __attribute__((aligned(256))) float s_stat0[2 * kRows], s_stat1[2 * kRows];
    __shared__ __attribute__((aligned(256))) u32x4 s_pass[kWaves][2][kWave];
    typedef typename T::vec8 vec8;

    const uint32_t id = work_of(blockIdx.x, a.blocks * a.parts * a.kv_heads);
    const uint32_t block = id % a.blocks;
    const uint32_t part = id / a.blocks % a.parts;
    const int bh = (int)(id / a.blocks / a.parts);
    const int b = bh / a.kv_heads, kvh = bh % a.kv_heads;
    const int lane = lane_id(), wave = wave_id(), half = lane >> 5;
    const int role = wave & 1;  // 0: rows 0 .. 31 of a tile, dv; 1: rows 32 .. 63, dk

    // with a mask, the block's keys are the next of the list
    const int at_key = (int)block * kPairHeld + (wave >> 1) * 32 + (lane & 31);
    const int keys = a.list ? a.counts[b] : admitted_keys(a, b);
    const bool valid = at_key < keys;
    const bool busy = ballot(valid) != 0;  // else a wave only loads and waits
    const int64_t key = a.list && valid ? a.list[(int64_t)b * a.keys + at_key] : at_key;
    f32x16 acc[DC / 32];
    clear(acc);
    float ds_scale = 1.0f;
    int t = (int)part * a.tiles_per_part, end = t + a.tiles_per_part;
    end = end < a.tiles ? end : a.tiles;

    if (__syncthreads_or(valid) && t < end) {
        const char* qbase = a.q + b * a.qb + (int64_t)kvh * a.group * a.qh;
        const char* gbase = g.d_o + b * g.dob + (int64_t)kvh * a.group * g.doh;
        // a wave each for the rows' two
        const char* stat_base =
            reinterpret_cast<const char*>(g.stat + (2 * (int64_t)bh + (wave & 1)) * a.rows);
        RowDma<DT, kRows> rq, rg;
        rq.init(qbase, a.ql, a.qh, a.group, a.dim, t);
        rg.init(gbase, g.dol, g.doh, a.group, a.dim, t);
        auto fetch = [&](char* to_q, char* to_g, float* to_stat) {
            const int left = a.rows - t * kRows;
            rq.issue(left, to_q);
            rg.issue(left, to_g);
            static_assert(kRows == kWave, "one load of a wave");
            if (wave < 2)
                dma4(buffer_at(stat_base + (int64_t)4 * kRows * t), lane < left ? 4 * lane : kOutside,
                     lds_address(to_stat + wave * kRows));
        };
        fetch(s_q0, s_g0, s_stat0);
        vec8 k[DC / 16], v[DC / 16];
        hold<T, DC>(k, a.k + b * a.kb + key * a.ks + kvh * a.kh, valid, a.dim);
        hold<T, DC>(v, a.v + b * a.vb + key * a.vs + kvh * a.vh, valid, a.dim);
        // with the 2^kGradShift that p carries taken out
        ds_scale = key_scale<T>(g, bh, v) * __builtin_ldexpf(1.0f, -(int)T::kGradShift);
        dma_wait();
        __syncthreads();
        auto step = [&](auto low, const char* tile_q, const char* tile_g, const float* stat,
                        char* next_q, char* next_g, float* next_stat) GSD_INLINE -> bool {
            constexpr bool kLow = decltype(low)::value;
            const bool more = ++t < end;
            if (more) {
                rq.next();
                rg.next();
                fetch(next_q, next_g, next_stat);
            }
            const int r0 = 32 * role;
            const char* mine = role ? tile_q : tile_g;  // what the sum's other factor is read from
            [[maybe_unused]] u32x4 pass_low[2];
            if (busy) {
                f32x16 s, dp;
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) {
                    // dp's sums begin at -delta
                    const f32x4 nd =
                        *reinterpret_cast<const f32x4*>(stat + kRows + r0 + 8 * i4 + 4 * half);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[4 * i4 + i] = 0.0f;
                        dp[4 * i4 + i] = nd[i];
                    }
                }
#pragma unroll
                for (int ks = 0; ks < DC / 16; ++ks) {
                    s = T::mma(read_rows<T, DT>(tile_q + r0 * DT * 2, 0, ks), k[ks], s);
                    dp = T::mma(read_rows<T, DT>(tile_g + r0 * DT * 2, 0, ks), v[ks], dp);
                }
                __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);  // -delta
                pace<DC / 16, 2, 2, 2>();
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) {
                    const f32x4 of = *reinterpret_cast<const f32x4*>(stat + r0 + 8 * i4 + 4 * half);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = 4 * i4 + i;
                        s[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], a.scale_log2, of[i]));
                        dp[j] = s[j] * (dp[j] * ds_scale);
                        if constexpr (kLow) dp[j] = formed(dp[j]);
                    }
                }
                vec8 keep[2], keep_low[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const vec8 p = pack<T>(s, j), ds = pack<T>(dp, j);
                    keep[j] = role ? ds : p;
                    s_pass[wave][j][lane] = __builtin_bit_cast(u32x4, role ? p : ds);
                    if constexpr (kLow) {
                        const vec8 p_low = pack_low<T>(s, j), ds_low = pack_low<T>(dp, j);
                        keep_low[j] = role ? ds_low : p_low;
                        pass_low[j] = __builtin_bit_cast(u32x4, role ? p_low : ds_low);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int db = 0; db < DC / 32; ++db) {
                        const vec8 with = read_columns<T, DT>(mine + r0 * DT * 2, 16 * j, db);
                        acc[db] = T::mma(with, keep[j], acc[db]);
                        if constexpr (kLow) acc[db] = T::mma(with, keep_low[j], acc[db]);
                    }
                if constexpr (!kLow) pace<DC / 16, 2, 1, 3>();
            }
            __syncthreads();
            auto add_passed = [&] {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const vec8 other = __builtin_bit_cast(vec8, s_pass[wave ^ 1][j][lane]);
#pragma unroll
                    for (int db = 0; db < DC / 32; ++db)
                        acc[db] = T::mma(read_columns<T, DT>(mine + (32 - r0) * DT * 2, 16 * j, db), other,
                                         acc[db]);
                }
                pace<DC / 16, 2, 1, 3>();
            };
            if (busy) add_passed();
            if constexpr (kLow) {
                // in the same place: with one more two work-groups would not fit a CU
                __syncthreads();
                if (busy)
#pragma unroll
                    for (int j = 0; j < 2; ++j) s_pass[wave][j][lane] = pass_low[j];
                __syncthreads();
                if (busy) add_passed();
            }
            if (more) {
                dma_wait();
                __syncthreads();
            }
            return more;
        };
        auto all = [&](auto low) GSD_INLINE {
            while (step(low, s_q0, s_g0, s_stat0, s_q1, s_g1, s_stat1) &&
                   step(low, s_q1, s_g1, s_stat1, s_q0, s_g0, s_stat0)) {
            }
        };
        if (!kFew && __builtin_expect(keys <= kFewTerms, 0))
            all(std::true_type{});
        else
            all(std::integral_constant<bool, kFew>{});
    }
    if (!valid) return;
    const float f = role ? a.scale / (ds_scale * __builtin_ldexpf(1.0f, (int)T::kGradShift))
                         : __builtin_ldexpf(1.0f, -(int)T::kGradShift);
    if (a.parts == 1) {
        const int64_t to = 2 * (((b * a.keys + key) * a.kv_heads + kvh) * (int64_t)a.dim);
        put<T, DC, false>(acc, f, (role ? g.dk : g.dv) + to, a.dim);
    } else {
        const int64_t to = (((int64_t)part * a.batch * a.kv_heads + bh) * a.keys + key) * a.dim;
        put<T, DC, true>(acc, f, (role ? g.partial_dk : g.partial_dv) + to, a.dim);
    }
}

// out = the parts' sums in order, for up to three gradients in one launch: eight
// values of a row per thread.  from [parts, batch kv_heads, rows, dim]; out [batch,
// rows / group, kv_heads, group, dim].
struct SumJob {
    const float* from;
    char* out;
    uint32_t parts, first_block;
    int32_t rows, group;
    int32_t of_keys;  // rows are keys: those that take no part have no sums
};
struct SumArgs {
    SumJob job[3];
    AttnArgs f;
    int32_t jobs, batch, kv_heads, dim;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void sum_parts_kernel(SumArgs a) {
    int k = 0;
    while (k + 1 < a.jobs && blockIdx.x >= a.job[k + 1].first_block) ++k;
    const SumJob j = a.job[k];
    const int units = a.dim / 8;
    const int64_t all = (int64_t)a.batch * a.kv_heads * j.rows;
    const int64_t id = (int64_t)(blockIdx.x - j.first_block) * kThreads + threadIdx.x;
    if (id >= all * units) return;
    const int64_t at = id / units;
    const int c = (int)(id - at * units);
    const int64_t bh = at / j.rows;
    const int row = (int)(at - bh * j.rows), l = row / j.group;
    const int64_t b = bh / a.kv_heads, kvh = bh - b * a.kv_heads;
    if (j.of_keys && !key_valid(a.f, b, row)) return;
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
    for (uint32_t p = 0; p < j.parts; ++p) {
        const float* x = j.from + (p * all + at) * a.dim + 8 * c;
        const f32x4 u = load_any<f32x4>(x), v = load_any<f32x4>(x + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc[i] += u[i];
            acc[4 + i] += v[i];
        }
    }
    const int64_t to = ((b * (j.rows / j.group) + l) * a.kv_heads + kvh) * j.group + (row - l * j.group);
    typename T::vec8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (typename T::elem)acc[i];
    store_any(j.out + 2 * (to * a.dim + 8 * c), o);
}

template <typename T>
hipError_t launch_typed(const GradArgs& base, const AttentionSplit& sq, const AttentionSplit& sk,
                        hipStream_t st) {
    const dim3 threads(kThreads);
    const int64_t heads = (int64_t)base.f.batch * base.f.kv_heads;
    auto split = [&](const AttentionSplit& s) {
        GradArgs g = base;
        g.f.blocks = (uint32_t)s.blocks;
        g.f.parts = (uint32_t)s.parts;
        g.f.total = (uint32_t)(s.blocks * s.parts * heads);
        g.f.tiles = (int32_t)s.tiles;
        g.f.tiles_per_part = (int32_t)((s.tiles + s.parts - 1) / s.parts);
        return g;
    };
    // without queries there are no rows: dk and dv are 0; without keys dq is
    auto run = [&](auto kernel, const GradArgs& g, int64_t groups) {
        if (groups > 0)
            hipLaunchKernelGGL(kernel, dim3((unsigned)groups), threads, 0, st, g);
    };
    const GradArgs gk = split(sk), gq = split(sq);
    const int64_t units = heads * base.f.keys * (base.f.dim / 8);
    const int64_t zero_groups =
        base.dk && (base.f.mask || base.f.lengths) ? (units + kThreads - 1) / kThreads : 0;
    const int64_t value_groups = T::kScaled ? heads * base.value_blocks : 0;
    run(delta_kernel<T>, base, heads * base.top_blocks + value_groups + zero_groups);
    if (base.f.list) {
        const hipError_t e = launch_key_list(base.f, st);
        if (e != hipSuccess) return e;
    }
    const int64_t key_groups = base.dk ? gk.f.total : 0, row_groups = base.dq ? gq.f.total : 0;
    auto run_dq = [&](auto dc, auto few) {
        constexpr int DC = decltype(dc)::value, DT = DC > 64 ? 128 : 64;
        constexpr bool kFew = decltype(few)::value;
        base.f.list ? run(dq_kernel<T, DT, DC, true, kFew>, gq, row_groups)
                    : run(dq_kernel<T, DT, DC, false, kFew>, gq, row_groups);
    };
    auto run_pairs = [&](auto dc) {
        constexpr int DC = decltype(dc)::value;
        few_terms(base.f.rows, base.f.keys) ? run(dkdv_pair_kernel<T, DC, true>, gk, key_groups)
                                            : run(dkdv_pair_kernel<T, DC, false>, gk, key_groups);
    };
    using Narrow = std::integral_constant<int, 64>;
    using Middle = std::integral_constant<int, kMiddle>;
    using Wide = std::integral_constant<int, 128>;
    const bool few = few_terms(base.f.rows, base.f.keys);
    if (base.f.dim <= 64) {
        few ? run(dkdv_kernel<T, 64, true>, gk, key_groups)
            : run(dkdv_kernel<T, 64, false>, gk, key_groups);
        few ? run_dq(Narrow{}, std::true_type{}) : run_dq(Narrow{}, std::false_type{});
    } else if (base.f.dim <= kMiddle) {
        run_pairs(Middle{});
        few ? run_dq(Middle{}, std::true_type{}) : run_dq(Middle{}, std::false_type{});
    } else {
        run_pairs(Wide{});
        few ? run_dq(Wide{}, std::true_type{}) : run_dq(Wide{}, std::false_type{});
    }
    SumArgs sum{};
    sum.f = base.f;
    sum.batch = base.f.batch;
    sum.kv_heads = base.f.kv_heads;
    sum.dim = base.f.dim;
    uint32_t sum_blocks = 0;
    auto add = [&](const float* from, char* out, int64_t parts, int64_t rows, int group) {
        if (parts <= 1 || !out) return;
        sum.job[sum.jobs++] = SumJob{from, out, (uint32_t)parts, sum_blocks, (int32_t)rows, group,
                                     out != base.dq};
        sum_blocks += (uint32_t)((heads * rows * (base.f.dim / 8) + kThreads - 1) / kThreads);
    };
    add(base.partial_dk, base.dk, sk.parts, base.f.keys, 1);
    add(base.partial_dv, base.dv, sk.parts, base.f.keys, 1);
    add(base.partial_dq, base.dq, sq.parts, base.f.rows, base.f.group);
    if (sum_blocks)
        hipLaunchKernelGGL(sum_parts_kernel<T>, dim3(sum_blocks), threads, 0, st, sum);
    return hipGetLastError();
}

}  // namespace

AttentionSplit attention_split_dq(const gsd_attention& g) {
    AttentionSplit s;
    s.blocks = (g.queries * (g.heads / g.kv_heads) + kHeld - 1) / kHeld;
    s.tiles = (g.keys + kTile - 1) / kTile;
    s.parts = split_parts(s.blocks * g.batch * g.kv_heads, s.tiles, 2, g.dim > 64 ? 2 : 4);
    return s;
}

AttentionSplit attention_split_dkdv(const gsd_attention& g) {
    AttentionSplit s;
    const int held = g.dim > 64 ? kPairHeld : kHeld;
    s.blocks = (g.keys + held - 1) / held;
    s.tiles = (g.queries * (g.heads / g.kv_heads) + kGradRows - 1) / kGradRows;
    s.parts = split_parts(s.blocks * g.batch * g.kv_heads, s.tiles, 2, g.dim > 64 ? 2 : 3);
    return s;
}

int64_t attention_top_blocks(const gsd_attention& g) {
    return (g.queries * (g.heads / g.kv_heads) + kDeltaRows - 1) / kDeltaRows;
}

int64_t attention_value_blocks(const gsd_attention& g) {
    return (g.keys + kDeltaRows - 1) / kDeltaRows;
}

hipError_t launch_attention_backward(const gsd_attention& a, const gsd_attention_grad& gr,
                                     const AttentionSplit& sq, const AttentionSplit& sk,
                                     const AttentionBackwardBuffers& buf, hipStream_t st) {
    GradArgs g{};
    g.f = attention_args(a, buf.list);
    g.d_o = static_cast<const char*>(gr.d_o);
    g.dob = 2 * gr.do_stride_b;
    g.dol = 2 * gr.do_stride_l;
    g.doh = 2 * gr.do_stride_h;
    g.stat = buf.stat;
    g.top = buf.top;
    g.top_blocks = (int32_t)attention_top_blocks(a);
    g.value_top = buf.value_top;
    // dq alone needs the values' norms
    g.value_blocks = gr.dq ? (int32_t)attention_value_blocks(a) : 0;
    g.dq = static_cast<char*>(gr.dq);
    g.dk = static_cast<char*>(gr.dk);
    g.dv = static_cast<char*>(gr.dv);
    g.partial_dq = buf.partial_dq;
    g.partial_dk = buf.partial_dk;
    g.partial_dv = buf.partial_dv;
    return a.dtype == GSD_BF16 ? launch_typed<Bf16>(g, sq, sk, st) : launch_typed<F16>(g, sq, sk, st);
}

}  // namespace gsd
