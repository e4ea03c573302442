// gsd_attention.h — what the attention kernels share: arguments, types of the
// matrix operands, the tile layout in LDS, and the valid keys of a tile.
//
// A batch and key head is one problem: its rows are the R = queries x (heads /
// kv_heads) pairs (query, query head), row r being query r / G of the group's
// head r % G, so the heads that share keys share every tile of them, and the
// sums of dk and dv over those heads are sums over rows.
//
// All products are 32x32x16 matrix instructions.  With l = lane % 32 and half =
// lane / 32, operand A holds row l and operand B column l, eight consecutive k
// from 8 half; the result holds column l and rows 8 (i / 4) + 4 half + i % 4 in
// its 16 registers i.  A product whose result is summed over its rows next is
// formed with those rows (keys in the forward and for dq, rows in dk and dv) as
// the result's rows: 16 values rounded to the type and packed in order are then
// operand B of that next product, in which k runs over rows 16 b + {4 half ..
// 4 half + 3, 8 + 4 half ..}.  Operand A is read in the same order with two
// transposing LDS reads, four consecutive rows each, so nothing passes through
// LDS between the two products.
#pragma once

#include <type_traits>

#include "gsd_common.h"
#include "gsd_internal.h"

namespace gsd {

// of a lambda whose captures live in registers
#define GSD_INLINE __attribute__((always_inline))

typedef short s16x4 __attribute__((ext_vector_type(4)));

// The forward's sums are scaled anew only where a row's maximum has grown by
// more than this power of two since they last were.
constexpr double kSlack = 8.0;

struct Bf16 {
    typedef __bf16 elem;
    typedef __bf16 vec8 __attribute__((ext_vector_type(8)));
    static constexpr float kShift = 0.0f, kGradShift = 0.0f;
    static constexpr bool kScaled = false;
    static __device__ __forceinline__ f32x16 mma(vec8 a, vec8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
struct F16 {
    typedef _Float16 elem;
    typedef _Float16 vec8 __attribute__((ext_vector_type(8)));
    // Below 2^-14 a 16-bit float loses bits, which the p of a few thousand
    // equal keys would reach in the backward, where p <= 1: it is formed as 2^15
    // p, and the factor taken out of the sums.  The forward's p = 2^(s - m) is at
    // most 2^kSlack; with 2^7 it stays below 2^15 as well.
    static constexpr float kShift = 7.0f, kGradShift = 15.0f;
    // ds = p (dp - delta) has the size of do times v: it is scaled by a power of two
    // from their norms, a row's for dq and a key's for dk
    static constexpr bool kScaled = true;
    static __device__ __forceinline__ f32x16 mma(vec8 a, vec8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

struct AttnArgs {
    const char *q, *k, *v;
    int64_t qb, ql, qh, kb, ks, kh, vb, vs, vh;  // strides, bytes
    const int32_t* lengths;
    const uint8_t* mask;
    int64_t mb, ms;
    // with a mask: the valid keys of each batch in order, and how many
    int32_t* list;
    int32_t* counts;
    char* o;
    char* o_low;  // o less its rounding, or null
    float* lse;
    int32_t rows;  // queries x group
    int64_t keys;
    int32_t batch, heads, kv_heads, group, dim;
    float scale, scale_log2;  // scale, scale log2 e
    float slack;              // kSlack in units of q.k
    // the grid: blocks x parts x (batch kv_heads)
    uint32_t blocks, parts, total;
    int32_t tiles, tiles_per_part;
    float* partial_o;
    float* partial_lse;
};

// Work-groups are dealt to the eight dies in turn.  Giving each pair of dies a
// consecutive share of a batch's work lets work-groups that walk the same keys or
// rows at once find them in their L2.  dk and dv of 4096 x 32400 with 16 heads of
// 128 in groups of 4 take 2.03 ms, 2.11 with a share for each die.  Each batch is
// shared out by itself, since lengths and masks differ: with 4134 and fewer keys
// for 1237 queries, 8 heads of 64 in groups of 4, o takes 34 and dq 39 us, 37 and
// 43 with shares of all batches' work.
__device__ __forceinline__ uint32_t work_of(uint32_t id, uint32_t batch_total) {
    const uint32_t before = id / batch_total * batch_total, in = id - before;
    const uint32_t share = batch_total / 4, rest = batch_total % 4;
    const uint32_t pair = in % 4, i = in / 4;
    return before + pair * share + (pair < rest ? pair : rest) + i;
}

// ---- tiles of 64 rows in LDS ----
// A row of DT elements is stored as chunks of 16 bytes, chunk c at place c ^
// swizzle(row), so that the lanes of a read meet different banks: those of
// read_rows take one chunk of 32 rows, those of read_columns two neighbouring
// chunks of four rows.  A read_columns instruction then costs 0.39 of a
// read_rows one (24 and 61 us for the same count of them on every CU); with the
// rows' low bits in the chunk's low bits it costs 0.57, and 7 times as much for
// read_rows without a swizzle.  Counters show no conflict for rows of 128; for rows of 64,
// whose swizzle has eight places instead of sixteen, conflicts are a quarter (dk and dv)
// to 0.4 (dq) of the LDS's cycles, and it is busy for 0.3 to 0.5 of the time.
constexpr int kTile = 64;

// p and ds are rounded to the type for their products: the errors average out over the
// sums' terms, to that of the result's own rounding.  Up to this many keys that take part
// (or rows, in dk and dv) they need not: one query and two keys give 2.5 times a result's
// own rounding.  What the rounding left out is then multiplied too.  A batch's keys count
// as its length or mask leaves them, not as they are padded.
constexpr int kFewTerms = 64;
static_assert(kFewTerms <= kTile, "so few keys are one tile");

// Heads up to 64 lie in rows of DT = 64, others in rows of 128.  Of those the products
// take DC elements: 96 where a head has no more, all 128 otherwise.  4096 x 32400, 16
// heads of 96 in groups of 4: o takes 0.83 ms and with its gradients 3.47, 0.92 and 3.97
// with products of 128; 2 x 1237 x 4134, 8 heads of 96: 52 and 245 us, 56 and 274.
constexpr int kMiddle = 96;

template <int DT>
__device__ __forceinline__ int swizzle(int row) {
    return DT == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : ((row & 3) << 1) | ((row >> 2) & 1);
}
template <int DT>
__device__ __forceinline__ int chunk_at(int row, int c) {
    return row * (DT / 8) + (c ^ swizzle<DT>(row));
}

// A product as its 32-bit value.  fp16 has an instruction that multiplies and rounds to
// 16 bits at once; with it in one of two places, the value that is stored and the one that
// is taken off to see what its rounding left out differ by a whole step now and then.
__device__ __forceinline__ float formed(float v) {
    asm("" : "+v"(v));
    return v;
}

// N values times f to o, what their rounding leaves out to o_low (or null).
template <typename T, int N>
__device__ __forceinline__ void put_rounded(char* o, char* o_low, int64_t at, const float (&v)[N],
                                            float f) {
    typedef typename T::elem vec __attribute__((ext_vector_type(N)));
    vec high, low;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float x = formed(v[i] * f);
        high[i] = (typename T::elem)x;
        low[i] = (typename T::elem)(x - (float)high[i]);
    }
    store_any(o + 2 * at, high);
    if (o_low) store_any(o_low + 2 * at, low);
}

// Operand A from a tile: rows r0 + l, elements 16 ks + 8 half .. + 7.
template <typename T, int DT>
__device__ __forceinline__ typename T::vec8 read_rows(const char* tile, int r0, int ks) {
    const int lane = lane_id();
    const int at = chunk_at<DT>(r0 + (lane & 31), 2 * ks + (lane >> 5));
    return *reinterpret_cast<const typename T::vec8*>(tile + 16 * at);
}

// Operand A from a tile read transposed: elements 32 db + l as rows, rows r0 +
// {4 half .. + 3, 8 + 4 half .. + 3} as k.  In each group of 16 lanes, lane i
// addresses 4 elements of row i / 4 and receives element i of four rows.
template <typename T, int DT>
__device__ __forceinline__ typename T::vec8 read_columns(const char* tile, int r0, int db) {
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    const int lane = lane_id();
    const int row = r0 + 4 * (lane >> 5) + ((lane >> 2) & 3);
    const int c = 4 * db + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
    const int in = 8 * (lane & 1);
    union {
        s16x4 h[2];
        typename T::vec8 v;
    } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_ptr)(tile + 16 * chunk_at<DT>(row, c) + in));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_ptr)(tile + 16 * chunk_at<DT>(row + 8, c) + in));
    return u.v;
}

// The order in which the compiler is to emit a run of products: `ahead` LDS
// reads first, then after every kMma products the reads of kRead more.  Left to
// itself it moves all reads to the front and runs out of registers.
template <int kSteps, int kRead, int kMma, int kAhead>
__device__ __forceinline__ void pace() {
    __builtin_amdgcn_sched_group_barrier(0x100, kRead * kAhead, 0);
#pragma unroll
    for (int i = 0; i < kSteps - kAhead; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, kMma, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, kRead, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kMma * kAhead, 0);
}

// The other half's v: lane l of one half receives lane l's of the other.
__device__ __forceinline__ float other_half(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    return __uint_as_float(lane_id() < 32 ? r[1] : r[0]);
}

// Eight results, registers 8 b .. 8 b + 7, as operand B.
template <typename T>
__device__ __forceinline__ typename T::vec8 pack(const f32x16& p, int b) {
    typename T::vec8 out;
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = (typename T::elem)p[8 * b + i];
    return out;
}

// What that rounding left out, rounded in its turn; p is `formed`.
template <typename T>
__device__ __forceinline__ typename T::vec8 pack_low(const f32x16& p, int b) {
    typename T::vec8 out;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        out[i] = (typename T::elem)(p[8 * b + i] - (float)(typename T::elem)p[8 * b + i]);
    return out;
}

// The keys that a batch's length admits.
__device__ __forceinline__ int admitted_keys(const AttnArgs& a, int b) {
    int n = (int)a.keys;
    if (a.lengths) {
        const int len = a.lengths[b];
        n = len < n ? len : n;
        n = n > 0 ? n : 0;
    }
    return n;
}

// Rows from memory straight to LDS: a wave's instruction moves 64 chunks of 16
// bytes to 1 KB of consecutive LDS, each lane naming the chunk that belongs
// there.  The lanes' offsets from a tile's first row are the same for every
// tile; chunks that are to be zero get an offset past the buffer's end, which
// reads as zero.
constexpr uint32_t kOutside = 0xfffffff0u;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

// A value that the compiler does not know: what depends on it is formed where it
// is used.
__device__ __forceinline__ int opaque(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

__device__ __forceinline__ uint32_t uniform(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}
__device__ __forceinline__ int wave_id() { return (int)uniform(threadIdx.x / kWave); }

// The buffer that starts at a uniform address, 2^31 bytes long.
__device__ __forceinline__ u32x4 buffer_at(const char* base) {
    const uint64_t p = reinterpret_cast<uint64_t>(base);
    return u32x4{uniform((uint32_t)p), uniform((uint32_t)(p >> 32)) & 0xffffu, 0x80000000u,
                 0x00020000u};
}

// N times sixteen bytes (one float) per lane, from the buffer's byte offset[i] to
// lds + 1024 i + 16 lane (lds + 4 lane).  The compiler does not see these loads:
// it would have every read of LDS wait for all of them, of other buffers too,
// and so for memory once per tile.  dma_wait() waits for those of the wave; a
// barrier behind it makes the work-group's visible.  The first s_nop covers the
// five states between a scalar register's write by a vector instruction and its
// use by a memory one, the others the one after a write of m0.  m0 is reserved: the
// compiler does not keep it over assembly that names it as changed (it warns there), so
// these kernels hold no other instruction that uses it.  kStream: data that is read once
// and not kept in the caches.
#define GSD_DMA16_X4(kind)                                                                   \
    asm volatile(                                                                            \
        "s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %5, 0 offen" kind " lds\n\t"   \
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"                                             \
        "buffer_load_dwordx4 %2, %5, 0 offen" kind " lds\n\t"                                \
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"                                             \
        "buffer_load_dwordx4 %3, %5, 0 offen" kind " lds\n\t"                                \
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"                                             \
        "buffer_load_dwordx4 %4, %5, 0 offen" kind " lds"                                    \
        :                                                                                    \
        : "s"(lds), "v"(offset[0]), "v"(offset[1]), "v"(offset[2]), "v"(offset[3]), "s"(buffer) \
        : "memory", "scc")
template <bool kStream = false, int N>
__device__ __forceinline__ void dma16(u32x4 buffer, const uint32_t (&offset)[N], uint32_t lds) {
    static_assert(N == 4 || (N == 2 && !kStream), "instructions per wave and tile");
    if constexpr (N == 2)
        asm volatile(
            "s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
            "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds"
            :
            : "s"(lds), "v"(offset[0]), "v"(offset[1]), "s"(buffer)
            : "memory", "scc");
    else if constexpr (kStream)
        GSD_DMA16_X4(" nt");
    else
        GSD_DMA16_X4("");
}
#undef GSD_DMA16_X4
__device__ __forceinline__ void dma4(u32x4 buffer, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :
                 : "s"(lds), "v"(offset), "s"(buffer)
                 : "memory");
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return uniform((uint32_t)reinterpret_cast<uintptr_t>(
        (const __attribute__((address_space(3))) void*)p));
}

template <int DT, int kRows = kTile>
struct TileDma {
    static constexpr int kChunks = kRows * DT / 8 / kThreads;  // instructions per wave
    uint32_t offset[kChunks];

    // The row and chunk that belong at a thread's place of instruction i.
    static __device__ __forceinline__ void place(int thread, int i, int& r, int& c) {
        const int at = (thread / kWave * kChunks + i) * kWave + thread % kWave;
        r = at / (DT / 8);
        c = at % (DT / 8) ^ swizzle<DT>(r);
    }
    // 0 <= stride < 2^25 bytes
    __device__ __forceinline__ void init(int64_t stride, int dim) {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            int r, c;
            place(threadIdx.x, i, r, c);
            offset[i] = 8 * c < dim ? (uint32_t)(r * stride) + 16 * c : kOutside;
        }
    }
    // left: rows from the tile's first on
    __device__ __forceinline__ void issue(const char* base, int left, char* tile) const {
        const u32x4 from = buffer_at(base);
        const uint32_t to = lds_address(tile) + wave_id() * kChunks * 1024;
        if (left >= kRows) {
            dma16(from, offset, to);
        } else {
            // formed here, where it is rare, and not held in registers for it
            const int thread = opaque(threadIdx.x);
            uint32_t some[kChunks];
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                int r, c;
                place(thread, i, r, c);
                some[i] = r < left ? offset[i] : kOutside;
            }
            dma16(from, some, to);
        }
    }
};

// The same for rows that a list names: lane l holds that of row l.
template <int DT>
struct ListDma {
    static constexpr int kChunks = TileDma<DT>::kChunks;
    uint32_t stride;
    int dim;
    __device__ __forceinline__ void init(int64_t s, int d) {
        stride = (uint32_t)s;
        dim = d;
    }
    // base: of the list's row 0; 0 <= row stride < 2^31 bytes
    __device__ __forceinline__ void issue(const char* base, int row, int left, char* tile) const {
        uint32_t offset[kChunks];
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            int r, c;
            TileDma<DT>::place(threadIdx.x, i, r, c);
            const uint32_t at = (uint32_t)__shfl(row, r) * stride + 16 * c;
            offset[i] = r < left && 8 * c < dim ? at : kOutside;
        }
        dma16(buffer_at(base), offset, lds_address(tile) + wave_id() * kChunks * 1024);
    }
};

// A walk over a part's tiles of keys, of the admitted ones or of a mask's list,
// whose rows are asked for one tile ahead.
template <bool kList>
struct KeyWalk {
    const int32_t* list;
    int n, t, end;
    int row, ahead;  // (list) the key of this lane's row of the tile, and of the next one

    __device__ __forceinline__ int ask(int tile) const {
        const int j = tile * kTile + lane_id();
        return j < n ? list[j] : 0;
    }
    __device__ __forceinline__ void start(const AttnArgs& a, int b, uint32_t part) {
        n = kList ? a.counts[b] : admitted_keys(a, b);
        if (kList) list = a.list + (int64_t)b * a.keys;
        const int last = (int)(((int64_t)n + kTile - 1) / kTile);
        // the tiles that there are, shared out evenly
        const int each = (last + (int)a.parts - 1) / (int)a.parts;
        t = (int)part * each;
        end = t + each < last ? t + each : last;
        if (kList && more()) row = ask(t);
    }
    __device__ __forceinline__ bool more() const { return t < end; }
    __device__ __forceinline__ int left() const { return n - t * kTile; }
    __device__ __forceinline__ void look_ahead() {
        if (kList && t + 1 < end) ahead = ask(t + 1);
    }
    __device__ __forceinline__ void next() {
        ++t;
        if (kList) row = ahead;
    }
};

// Keys and values of the walk's tile on their way to LDS.
template <bool kList, int DT>
struct KeyDma {
    typename std::conditional<kList, ListDma<DT>, TileDma<DT>>::type k, v;
    const char *kbase, *vbase;
    int64_t ks, vs;
    __device__ __forceinline__ void init(const AttnArgs& a, int b, int kvh) {
        kbase = a.k + b * a.kb + kvh * a.kh;
        vbase = a.v + b * a.vb + kvh * a.vh;
        ks = a.ks;
        vs = a.vs;
        k.init(ks, a.dim);
        v.init(vs, a.dim);
    }
    __device__ __forceinline__ void fetch(const KeyWalk<kList>& w, char* to_k, char* to_v) const {
        if constexpr (kList) {
            k.issue(kbase, w.row, w.left(), to_k);
            v.issue(vbase, w.row, w.left(), to_v);
        } else {
            k.issue(kbase + (int64_t)w.t * kTile * ks, w.left(), to_k);
            v.issue(vbase + (int64_t)w.t * kTile * vs, w.left(), to_v);
        }
    }
};

// Whether result register i of sub-tile h is a key past the last; `lane` opaque, so
// that what only a last tile needs is not held for all of them.
__device__ __forceinline__ bool past(int h, int i, int lane, int left) {
    return 32 * h + 8 * (i / 4) + i % 4 >= left - 4 * (lane >> 5);
}

}  // namespace gsd
