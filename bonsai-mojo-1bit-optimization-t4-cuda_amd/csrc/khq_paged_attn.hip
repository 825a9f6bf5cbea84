// khq_paged_attn.hip -- attention of new tokens over a paged cache.
//
// The rows of one KV head of a sequence, row r = query token r / n_rep, head
// r % n_rep of its group, are cut into row tiles, and where those are fewer
// than the chip's blocks, a tile's keys into splits whose partial results
// (unnormalised sum, maximum, sum of weights) a second launch joins in order.
// Everything about lengths is read on the device, so a captured launch follows
// them: each wavefront derives the whole partition from cu_q and seq_kv again
// (schedule below), which for one sequence is a few scalar operations and for
// some hundred one pass of a wavefront, about a microsecond.
//
// Row tiles come in two sizes: up to 16 rows of a sequence (a decode step's 6 of
// 24 / 4 heads), and all rows of a light batch, stream keys and values through
// registers (stream_item); more go in tiles of 128 or 256 rows that share keys
// and values in LDS (tile_item).  One launch serves both, or the first alone.
#include "khq_mfma_util.h"
#include "khq_paged_internal.h"

#include <algorithm>
#include <type_traits>

namespace khq {
namespace paged {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
// the caller's rows: any address of a 16-bit element
typedef uint32_t u4e __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u2e __attribute__((ext_vector_type(2), aligned(2)));

template <typename T>
struct V {
    typedef T x2 __attribute__((ext_vector_type(2)));
    typedef T x4 __attribute__((ext_vector_type(4)));
    typedef T x8 __attribute__((ext_vector_type(8)));
};
__device__ __forceinline__ f4 mfma16(V<fp16>::x8 a, V<fp16>::x8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f4 mfma16(V<bf16>::x8 a, V<bf16>::x8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16v mfma32(V<fp16>::x8 a, V<fp16>::x8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16v mfma32(V<bf16>::x8 a, V<bf16>::x8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// Two floats rounded to the type (to nearest even).
template <typename T>
__device__ __forceinline__ uint32_t pack(float x, float y) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{x, y}, typename V<T>::x2));
}
// l plus the two values of a packed pair.
template <typename T>
__device__ __forceinline__ float add_pair(uint32_t p, float l) {
    typedef typename V<T>::x2 x2;
    const x2 v = __builtin_bit_cast(x2, p);
    if constexpr (__is_same(T, fp16)) {
        return __builtin_amdgcn_fdot2(v, x2{(T)1.0f, (T)1.0f}, l, false);
    } else {
        return l + ((float)v[0] + (float)v[1]);
    }
}
// A pair with infinities and NaN as the type's largest values: a weight of 0
// makes a 0 of them.
template <typename T>
__device__ __forceinline__ uint32_t finite_pair(uint32_t p) {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    const unsigned short top = __is_same(T, fp16) ? 0x7bff : 0x7f7f;
    const us2 size = __builtin_elementwise_min(__builtin_bit_cast(us2, p & 0x7fff7fffu), us2{top, top});
    return (p & 0x80008000u) | __builtin_bit_cast(uint32_t, size);
}
template <typename T>
__device__ __forceinline__ bool nonfinite_pair(uint32_t p) {
    return finite_pair<T>(p) != p;
}
template <typename T>
__device__ __forceinline__ float sigmoid(T g) {
    return __builtin_amdgcn_rcpf(1.0f + __expf(-(float)g));  // each to a unit of 2^-23
}

// Reference maximum of a row that has seen no key: finite, so that a masked
// score (-inf) less it is -inf and its weight 0 without a test.
constexpr float M_NONE = -1e30f;
constexpr float LOG2E = 1.44269504f;
// A row's reference rises only when a score passes it by this (in log2 units):
// weights stay below e^10, far from the type's largest value.
constexpr float GAP = 10.0f * LOG2E;

// Scores in log2 units, so that a weight is one exp2; not 0, whose product
// with a masked score would be no number.
__device__ __forceinline__ float score_scale(float scale) {
    const float s = fmaxf(fabsf(scale) * LOG2E, 1e-30f);
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(s)));  // a scalar register's
}

// ------------------------------------------------------------ the partition
constexpr int SMALL_ROWS = 16;
// Blocks of the stream kernel: 4 wavefronts, two blocks a CU; 8 and one where
// they share a launch with tiles.  A unit is a 32-key tile for each wavefront.
constexpr int STREAM_WAVES = 4, STREAM_SLOTS = 512;
constexpr int TILE_UNIT = 64;

// Which sequences a launch serves: by their rows, or all of them.
enum Serve { SERVE_SMALL, SERVE_LARGE, SERVE_ALL };

struct Part {
    int rows;   // of a row tile
    int unit;   // keys
    int slots;  // blocks
    int room;   // of them, what the cost is shared among where items are nearly as many
    Serve serve;
    size_t at;  // of its partial results in the workspace, in floats
};

struct Item {
    int seq, row0, n_q, kv;  // sequence, its first batch row, rows and tokens
    int head, qt, split, n_split;
    int part;  // partial result of split 0 where there are several; of split i: part + i * H_kv
};

struct SeqLen {
    int row0, n_q, kv, tiles, units;  // tiles: row tiles (0: not served)
};

__device__ __forceinline__ SeqLen seq_len(const AttnArgs& a, const Part& pt, int s) {
    SeqLen l;
    const int c0 = a.r.cu_q[s], c1 = min(a.r.cu_q[s + 1], a.r.n_tok);
    l.row0 = c0;
    l.n_q = c0 >= 0 ? max(c1 - min(c0, a.r.n_tok), 0) : 0;  // none from outside the batch
    l.kv = min(max(a.r.seq_kv[s], 0), a.r.table_ld * a.p.page_size);
    const int rows = l.n_q * a.n_rep;
    const bool mine = pt.serve == SERVE_ALL || (rows <= SMALL_ROWS) == (pt.serve == SERVE_SMALL);
    l.tiles = mine ? (rows + pt.rows - 1) / pt.rows : 0;
    // units of the middle row: what a tile costs on average
    l.units = max(1, (max(l.kv - l.n_q / 2, 0) + pt.unit - 1) / pt.unit);
    return l;
}

// Inclusive sums over the lanes: within rows of 16, then rows to the right of
// lanes 15, 31 and 47.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_from(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int as_bits(int v) { return v; }
__device__ __forceinline__ int as_bits(float v) { return __float_as_int(v); }
template <typename T>
__device__ __forceinline__ T scan_add(T v) {
    auto of = [](int x) { return __builtin_bit_cast(T, x); };
    v += of(dpp_from<0x111, 0xF>(as_bits(v)));  // row_shr 1, 2, 4, 8
    v += of(dpp_from<0x112, 0xF>(as_bits(v)));
    v += of(dpp_from<0x114, 0xF>(as_bits(v)));
    v += of(dpp_from<0x118, 0xF>(as_bits(v)));
    v += of(dpp_from<0x142, 0xA>(as_bits(v)));  // row_bcast 15, 31
    v += of(dpp_from<0x143, 0xC>(as_bits(v)));
    return v;
}
template <typename T>
__device__ __forceinline__ T lane63(T v) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(as_bits(v), 63));
}

// The partition: items (row tile of a KV head) and what they are split into.
// Items are numbered sequence by sequence, with LONG (and up to 64 sequences)
// those of the longest blocks first; within a sequence, KV heads in turn
// (blocks go to the XCDs in turn, so a head's row tiles meet its keys in one
// L2), then splits, then row tiles from the last, which sees most keys, to the
// first.  A block takes at most u units.  With items few beside the slots
// u = cost / (slots - items): sum of ceil(units / u) <= cost / u + items <=
// slots, one round of blocks.  With more, cost / room, and from the slots' own
// number on cost / slots: alike items stay whole, one of a long sequence among
// short ones does not outlast the others.  Partial
// results: at most 2 cost / u <= 2 slots, as an item that is split has more
// than u units.  (The cost is a float sum, taken a little larger.)
struct Schedule {
    SeqLen one;          // this lane's sequence, where they are at most 64
    int per, u;          // sequences a lane, units a block
    int at, part;        // items and partial results before this lane's sequences
    int n_item, total;   // items of this lane's sequences, and of all
};
__device__ __forceinline__ int splits_of(const Schedule& sc, const SeqLen& l) {
    return l.units <= sc.u ? 1 : (int)ceilf((float)l.units / (float)sc.u);
}
// (64 lanes' stay in 31 bits: a batch within the sizes has 2^23, but cu_q may
// name the same rows for many sequences)
constexpr int MOST_ITEMS = 1 << 24;
template <bool LONG>
__device__ __forceinline__ Schedule schedule(const AttnArgs& a, const Part& pt, bool joining) {
    const int lane = threadIdx.x & 63, n_seq = a.r.n_seq, h_kv = a.p.H_kv;
    Schedule sc;
    sc.per = (n_seq + 63) >> 6;
    const int s0 = lane * sc.per, s1 = min(s0 + sc.per, n_seq);
    sc.one = SeqLen{};
    int items = 0;
    float cost = 0.0f;
    for (int s = s0; s < s1; s++) {
        sc.one = seq_len(a, pt, s);
        items = min(items + sc.one.tiles * h_kv, MOST_ITEMS);
        cost += (float)(sc.one.tiles * h_kv) * (float)sc.one.units;
    }
    const int all = lane63(scan_add(items));
    const int room = all >= pt.slots ? pt.slots : max(pt.slots - all, pt.room);
    const float share = lane63(scan_add(cost)) * 1.00001f / (float)room;
    sc.u = max(1, (int)fminf(ceilf(share), 1e9f));
    int n_part = 0, longest = 0;
    sc.n_item = 0;
    for (int s = s0; s < s1; s++) {
        if (sc.per > 1) sc.one = seq_len(a, pt, s);
        const int n = sc.one.tiles * h_kv, sp = splits_of(sc, sc.one);
        n_part += sp > 1 ? n * sp : 0;
        sc.n_item = min(sc.n_item + (joining ? (sp > 1 ? n : 0) : n * sp), MOST_ITEMS);
        if (LONG) longest = (int)((float)sc.one.units / (float)sp);
    }
    sc.at = scan_add(sc.n_item);
    sc.total = lane63(sc.at);
    sc.at -= sc.n_item;
    sc.part = scan_add(n_part) - n_part;
    if (LONG && sc.per == 1 && n_seq > 1) {
        sc.at = 0;
        for (int j = 0; j < n_seq; j++) {
            const int other = __builtin_amdgcn_readlane(longest, j), n = __builtin_amdgcn_readlane(sc.n_item, j);
            sc.at += other > longest || (other == longest && j < lane) ? n : 0;
        }
    }
    return sc;
}
// Row tile, from the last, that is started q-th of a lone sequence's.  Longest
// first, each round of blocks (w tiles of every head) ends the rounds before it
// evenly: a block that took the longest gets the shortest.  So an even number of
// rounds ends as one; of an odd number the last one starts as one and ends
// unevenly (a prompt of 8,192, 24 heads of 256, is 3: a tenth of the chip idle).
// There the round before it takes every other tile first, then the others: the
// blocks then come free spread as the last round's tiles are long.
__device__ __forceinline__ int started(const AttnArgs& a, const Part& pt, int q, int tiles) {
    const int w = a.by_kv.div(pt.slots);
    if (tiles <= 2 * w || w < 2) return q;
    const int rounds = (int)((uint32_t)(tiles + w - 1) / (uint32_t)w), i = q - (rounds - 2) * w, half = (w + 1) >> 1;
    if (rounds % 2 == 0 || i < 0 || i >= w) return q;
    return q - i + (i < half ? 2 * i : 2 * (i - half) + 1);
}
// Item x, below sc.total.
__device__ __forceinline__ Item item_of(const AttnArgs& a, const Part& pt, const Schedule& sc, int x,
                                        bool joining) {
    const int lane = threadIdx.x & 63, h_kv = a.p.H_kv;
    const unsigned long long has = __ballot(sc.at <= x && x < sc.at + sc.n_item);
    const int owner = __ffsll(has) - 1;
    SeqLen one = sc.one;
    int at = sc.at, part = sc.part, seq = lane * sc.per;
    if (sc.per > 1 && lane == owner) {  // the owner walks its sequences
        const int s1 = min(seq + sc.per, a.r.n_seq);
        for (int s = seq; s < s1; s++) {
            one = seq_len(a, pt, s);
            seq = s;
            const int n = one.tiles * h_kv, sp = splits_of(sc, one);
            const int c = joining ? (sp > 1 ? n : 0) : n * sp;
            if (x < at + c) break;
            at += c;
            part += sp > 1 ? n * sp : 0;
        }
    }
    auto from = [&](int v) { return __builtin_amdgcn_readlane(v, owner); };
    Item it;
    it.seq = from(seq);
    it.row0 = from(one.row0);
    it.n_q = from(one.n_q);
    it.kv = from(one.kv);
    it.n_split = from(splits_of(sc, one));
    const int tiles = from(one.tiles), j = x - from(at), k = a.by_kv.div(j);
    it.head = j - k * h_kv;
    const int q = joining || it.n_split == 1 ? k : (int)((uint32_t)k / (uint32_t)it.n_split);
    it.split = joining ? 0 : k - q * it.n_split;
    const bool lone = a.r.n_seq == 1 && it.n_split == 1;
    it.qt = tiles - 1 - (lone ? started(a, pt, q, tiles) : q);  // row tiles from the last
    it.part = from(part) + q * it.n_split * h_kv + it.head;
    return it;
}
// Units [lo, hi) of the item's split, of `units`: the first ones have one more.
__device__ __forceinline__ void split_units(const Item& it, int units, int& lo, int& hi) {
    lo = 0;
    hi = units;
    if (it.n_split == 1) return;
    const int each = (int)((uint32_t)units / (uint32_t)it.n_split), more = units - each * it.n_split;
    lo = each * it.split + min(it.split, more);
    hi = lo + each + (it.split < more ? 1 : 0);
}

// Tokens that row r of the item's sequence sees.
__device__ __forceinline__ int visible(const AttnArgs& a, const Item& it, int r) {
    return min(it.kv, max(0, it.kv - it.n_q + a.by_rep.div(r) + 1));
}
// Element offset of token t of a sequence in the pages (0 and bad set for a
// table entry outside the cache).
__device__ __forceinline__ long long token_at(const AttnArgs& a, const Item& it, int t, bool& bad) {
    const int pg = a.by_page.div(t), in = t - pg * a.p.page_size;
    int e = a.r.table[(size_t)it.seq * a.r.table_ld + pg];
    bad = (unsigned)e >= (unsigned)a.p.n_pages;
    e = bad ? 0 : e;
    return e * a.p.page_stride + in * a.p.token_stride + it.head * a.p.head_stride;
}

// Partial results: f32 [2 slots][rows][D] (each kernel's own order of one's
// values), then (maximum, sum) f32 pairs [2 slots][rows].
__device__ __forceinline__ float* part_acc(const AttnArgs& a, const Part& pt, int d, int part) {
    return static_cast<float*>(a.r.ws) + pt.at + (size_t)part * pt.rows * d;
}
__device__ __forceinline__ float2* part_ml(const AttnArgs& a, const Part& pt, int d, int part) {
    return reinterpret_cast<float2*>(static_cast<float*>(a.r.ws) + pt.at + (size_t)2 * pt.slots * pt.rows * d) +
           (size_t)part * pt.rows;
}

// x, of which the compiler knows nothing: what follows from it is computed where
// it is used, and not kept in registers that there are not.
__device__ __forceinline__ int opaque(int x) {
    asm("" : "+v"(x));
    return x;
}
__device__ __forceinline__ long long uniform(long long x) {
    const int lo = __builtin_amdgcn_readfirstlane((int)x), hi = __builtin_amdgcn_readfirstlane((int)(x >> 32));
    return ((long long)hi << 32) | (uint32_t)lo;
}

// ------------------------------------------------------------ few rows
// A wavefront takes 32-key tiles by itself, 16 rows on 16x16x32 MFMAs.  MFMA
// operands come straight from global loads: S^T = K Q^T takes K rows as they
// lie (lane: key, 8 dims); its result (row = lane % 16, keys 4 (lane / 16) + r
// of both 16-key halves) is the B operand of O^T += V^T P^T when that
// product's K index 8 g + j stands for key 4 g + j (j < 4) and 16 + 4 g + j - 4;
// a lane loads those 8 keys' values of 8 consecutive dims and transposes them
// in its registers (32 byte permutes), dim 8 m + t standing for row m of
// product t.  No LDS and no barrier until the block's wavefronts join.  Bound:
// memory; what it takes is loads under way, so a tile's 32 of 16 bytes are all
// issued before the first product, 256 registers a lane and two blocks of 4 a
// CU.  24 / 4 heads of 256 in fp16: 32 sequences of 1K to 16K tokens, 680 MB in
// 130 us (5.2 TB/s; a copy of 2 GB runs at 4.9), one of 131,071, 537 MB in 98
// (5.5); 512 tokens, of which latency is all, 8.6.
template <typename T, int D, int NW>
__device__ __forceinline__ void stream_item(const AttnArgs& a, const Part& pt, const Item& it, char* smem) {
    constexpr int KS = D / 32;                             // K steps of a score
    constexpr int VE = D == 64 ? 4 : 8, NH = D / 16 / VE;  // dims a lane loads at once, times
    constexpr int LD = D + 4;
    typedef typename V<T>::x8 x8;
    struct Lds {
        float acc[NW][16][LD], m[NW][16], l[NW][16];
        T q[16][D + 8];
    };
    Lds& lds = *reinterpret_cast<Lds*>(smem);
    const int tid = threadIdx.x, wv = tid >> 6, lane = tid & 63, li = lane & 15, lg = lane >> 4;
    const int rows = min(16, it.n_q * a.n_rep - it.qt * 16);  // of this tile
    const int r0 = it.qt * 16;
    // ---- queries into LDS, the scale's sign with them
    const uint32_t flip = a.r.scale < 0.0f ? 0x80008000u : 0u;
    for (int i = tid; i < 16 * (D / 8); i += 64 * NW) {
        const int row = i / (D / 8), c = i % (D / 8);
        u4e v = {0u, 0u, 0u, 0u};
        if (row < rows) {
            const int r = r0 + row, tok = a.by_rep.div(r), hq = it.head * a.n_rep + r - tok * a.n_rep;
            v = *reinterpret_cast<const u4e*>((const T*)a.r.q + (it.row0 + tok) * a.r.q_token +
                                              hq * a.r.q_head + 8 * c);
        }
        *reinterpret_cast<u4*>(&lds.q[row][8 * c]) = u4{v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip};
    }
    __syncthreads();
    // (256 dims: 32 registers of them, and as many too few for all of a tile's
    // loads at once; they are read again for each tile)
    x8 qf[KS];
    auto read_q = [&]() {
        const T* q = &lds.q[0][0] + opaque(li * (D + 8) + 8 * lg);
#pragma unroll
        for (int st = 0; st < KS; st++) qf[st] = *reinterpret_cast<const x8*>(q + 32 * st);
    };
    if (D < 256) read_q();
    const int vis = visible(a, it, r0 + min(li, rows - 1));  // (no row: what the last one sees)
    const int vis_lo = visible(a, it, r0), vis_hi = visible(a, it, r0 + rows - 1);
    const int units = (vis_hi + 32 * NW - 1) / (32 * NW);
    int t_lo, t_hi;
    split_units(it, units, t_lo, t_hi);
    t_lo *= NW;
    t_hi = min(t_hi * NW, (vis_hi + 31) >> 5);
    const float sc2 = score_scale(a.r.scale);
    const T* kp = (const T*)a.p.k;
    const T* vp = (const T*)a.p.v;
    f4 acc[NH][VE];
#pragma unroll
    for (int h = 0; h < NH; h++)
#pragma unroll
        for (int t = 0; t < VE; t++) acc[h][t] = f4{0.f, 0.f, 0.f, 0.f};
    float m_ref = M_NONE, l_part = 0.0f;
    // The block table's entries are read a tile ahead.  In pages of a multiple of
    // 32 tokens a tile lies in one: addresses are a scalar and 32 bits of a lane's.
    const bool by_tile = a.p.page_size % 32 == 0 && a.p.token_stride * a.p.page_size < 1 << 28;
    const int last = vis_hi - 1, ts = (int)a.p.token_stride;
    auto entry_of = [&](int t) {
        return a.r.table[(size_t)it.seq * a.r.table_ld + a.by_page.div(min(t * 32 + (lane & 31), last))];
    };
    int entry = t_lo + wv < t_hi ? entry_of(t_lo + wv) : 0;
    for (int t = t_lo + wv; t < t_hi; t += NW) {
        const int key0 = t * 32;
        // a lane's key: tokens past the last one seen stand for it
        const int tok = min(key0 + (lane & 31), last), in = tok - a.by_page.div(tok) * a.p.page_size;
        const bool bad = (unsigned)entry >= (unsigned)a.p.n_pages;
        const unsigned long long bad_keys = __ballot(bad);
        const int page = bad ? 0 : entry;
        const long long off = page * a.p.page_stride + in * a.p.token_stride + it.head * a.p.head_stride;
        if (t + NW < t_hi) entry = entry_of(t + NW);
        u4 kr[2][KS];
        uint32_t vr[8][NH][VE / 2];
        auto loads = [&](auto k_row, auto v_row) __attribute__((always_inline)) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const T* src = k_row(16 * h + li);
#pragma unroll
                for (int st = 0; st < KS; st++) kr[h][st] = *reinterpret_cast<const u4*>(src + 32 * st);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const T* src = v_row((j & 4) * 4 + 4 * lg + (j & 3));
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    if constexpr (VE == 8) {
                        const u4 v = *reinterpret_cast<const u4*>(src + 128 * h);
                        vr[j][h][0] = v.x; vr[j][h][1] = v.y; vr[j][h][2] = v.z; vr[j][h][3] = v.w;
                    } else {
                        const u2 v = *reinterpret_cast<const u2*>(src);
                        vr[j][h][0] = v.x; vr[j][h][1] = v.y;
                    }
                }
            }
        };
        if (by_tile) {
            const long long at = uniform(off);  // of the tile's first key, lane 0's
            const int most = last - key0;
            loads([&](int k) { return kp + at + (uint32_t)(min(k, most) * ts + 8 * lg); },
                  [&](int k) { return vp + at + (uint32_t)(min(k, most) * ts + VE * li); });
        } else {
            loads([&](int k) { return kp + __shfl(off, k, 64) + 8 * lg; },
                  [&](int k) { return vp + __shfl(off, k, 64) + VE * li; });
        }
        __builtin_amdgcn_sched_barrier(0);  // all loads on their way before the first product waits
        if (D == 256) read_q();
        f4 s[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            s[h] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < KS; st++) s[h] = mfma16(__builtin_bit_cast(x8, kr[h][st]), qf[st], s[h]);
        }
        // ---- mask: keys 16 h + 4 lg + r of row li
        float sc[8];
#pragma unroll
        for (int e = 0; e < 8; e++) sc[e] = s[e >> 2][e & 3];
        if (bad_keys) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (bad_keys >> (16 * (e >> 2) + 4 * lg + (e & 3)) & 1) sc[e] = __builtin_nanf("");
        }
        bool odd = false;  // values that are no numbers where a row's mask has to hold
        if (key0 + 32 > vis_lo) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (key0 + 16 * (e >> 2) + 4 * lg + (e & 3) >= vis) sc[e] = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const bool none = key0 + (j & 4) * 4 + 4 * lg + (j & 3) >= vis_hi;
#pragma unroll
                for (int h = 0; h < NH; h++)
#pragma unroll
                    for (int w = 0; w < VE / 2; w++) {
                        if (none) vr[j][h][w] = 0u;
                        odd = odd || nonfinite_pair<T>(vr[j][h][w]);
                    }
            }
            odd = __ballot(odd) != 0ull;
        }
        // ---- running maximum, raised only when it must be
        float lmax = sc[0];
#pragma unroll
        for (int e = 1; e < 8; e++) lmax = fmaxf(lmax, sc[e]);
        lmax *= sc2;
        if (__ballot(lmax > m_ref + GAP) != 0ull) {
            lmax = fmaxf(lmax, __shfl_xor(lmax, 16, 64));
            lmax = fmaxf(lmax, __shfl_xor(lmax, 32, 64));
            const float m_new = fmaxf(m_ref, lmax);
            const float fac = __builtin_amdgcn_exp2f(m_ref - m_new);  // 0 from M_NONE, 1 where it stays
            m_ref = m_new;
            l_part *= fac;
#pragma unroll
            for (int h = 0; h < NH; h++)
#pragma unroll
                for (int e = 0; e < VE; e++) acc[h][e] *= fac;
        }
        uint32_t pw[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            pw[e] = pack<T>(__builtin_amdgcn_exp2f(fmaf(sc[2 * e], sc2, -m_ref)),
                            __builtin_amdgcn_exp2f(fmaf(sc[2 * e + 1], sc2, -m_ref)));
            l_part = add_pair<T>(pw[e], l_part);
        }
        const x8 pb = __builtin_bit_cast(x8, u4{pw[0], pw[1], pw[2], pw[3]});
        if (odd) {
            // 0 * inf is no 0: such values leave the product and join the rows that see them
            for (int k = 0; k < 32; k++) {
                const T* src = vp + __shfl(off, k, 64);
                const bool sees = key0 + k < vis;
#pragma unroll
                for (int h = 0; h < NH; h++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
#pragma unroll
                        for (int e = 0; e < VE; e++) {
                            const float v = (float)src[VE * 16 * h + VE * (4 * lg + r) + e];
                            acc[h][e][r] += sees && !(fabsf(v) < INFINITY) ? v : 0.0f;
                        }
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int h = 0; h < NH; h++)
#pragma unroll
                    for (int w = 0; w < VE / 2; w++) vr[j][h][w] = finite_pair<T>(vr[j][h][w]);
        }
#pragma unroll
        for (int h = 0; h < NH; h++)
#pragma unroll
            for (int e = 0; e < VE; e++) {
                uint32_t w[4];
                const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    w[i] = __builtin_amdgcn_perm(vr[2 * i + 1][h][e >> 1], vr[2 * i][h][e >> 1], sel);
                acc[h][e] = mfma16(__builtin_bit_cast(x8, u4{w[0], w[1], w[2], w[3]}), pb, acc[h][e]);
            }
    }
    // ---- the wavefronts join in LDS
    l_part += __shfl_xor(l_part, 16, 64);
    l_part += __shfl_xor(l_part, 32, 64);
    if (lg == 0) {
        lds.m[wv][li] = m_ref;
        lds.l[wv][li] = l_part;
    }
#pragma unroll
    for (int h = 0; h < NH; h++)
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int e = 0; e < VE; e += 4)
                *reinterpret_cast<f4*>(&lds.acc[wv][li][VE * 16 * h + VE * (4 * lg + r) + e]) =
                    f4{acc[h][e][r], acc[h][e + 1][r], acc[h][e + 2][r], acc[h][e + 3][r]};
    __syncthreads();
    const bool direct = it.n_split == 1;
    const int part = it.part + it.split * a.p.H_kv;
    for (int i = tid; i < rows * (D / 4); i += 64 * NW) {
        const int row = i / (D / 4), c = (i % (D / 4)) * 4;
        float m = lds.m[0][row];
#pragma unroll
        for (int w = 1; w < NW; w++) m = fmaxf(m, lds.m[w][row]);
        f4 o = {0.f, 0.f, 0.f, 0.f};
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = __builtin_amdgcn_exp2f(lds.m[w][row] - m);
            o += *reinterpret_cast<const f4*>(&lds.acc[w][row][c]) * f;
            l += lds.l[w][row] * f;
        }
        if (direct) {
            const int r = r0 + row, tok = a.by_rep.div(r), hq = it.head * a.n_rep + r - tok * a.n_rep;
            const float inv = visible(a, it, r) > 0 ? 1.0f / l : 0.0f;
            o *= inv;
            if (a.r.gate) {
                const u2e g = *reinterpret_cast<const u2e*>(
                    (const T*)a.r.gate + (it.row0 + tok) * a.r.gate_token + hq * a.r.gate_head + c);
                const typename V<T>::x4 gv = __builtin_bit_cast(typename V<T>::x4, u2{g.x, g.y});
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] *= sigmoid(gv[e]);
            }
            *reinterpret_cast<u2e*>((T*)a.r.out + (it.row0 + tok) * a.r.out_token + hq * a.r.out_head + c) =
                u2e{pack<T>(o[0], o[1]), pack<T>(o[2], o[3])};
        } else {
            *reinterpret_cast<f4*>(part_acc(a, pt, D, part) + row * D + c) = o;
            if (c == 0) part_ml(a, pt, D, part)[row] = float2{m, l};
        }
    }
}

// The splits of row `row` of an item: a block's JW wavefronts sum every JW-th
// and meet in LDS, each with eight splits and their maxima in flight.
template <typename T, int D, int JW>
__device__ __forceinline__ void stream_join(const AttnArgs& a, const Part& pt, const Item& it, int row) {
    constexpr int E = D / 64;  // dims a lane
    typedef float fe __attribute__((ext_vector_type(E)));
    __shared__ float s_o[JW][D];
    __shared__ float2 s_ml[JW];
    const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63, h_kv = a.p.H_kv, r = it.qt * 16 + row;
    fe o = {};
    float m = M_NONE, l = 0.0f;
    for (int i0 = wv; i0 < it.n_split; i0 += 8 * JW) {
        float2 ml[8];
        fe v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int i = min(i0 + JW * j, it.n_split - 1);
            ml[j] = part_ml(a, pt, D, it.part + i * h_kv)[row];
            v[j] = *reinterpret_cast<const fe*>(part_acc(a, pt, D, it.part + i * h_kv) + row * D + E * lane);
        }
        float top = m;
#pragma unroll
        for (int j = 0; j < 8; j++) top = fmaxf(top, ml[j].x);
        const float f0 = __builtin_amdgcn_exp2f(m - top);
        m = top;
        l *= f0;
        o *= f0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (i0 + JW * j >= it.n_split) break;
            const float f = __builtin_amdgcn_exp2f(ml[j].x - m);
            l += ml[j].y * f;
            o += v[j] * f;
        }
    }
    __syncthreads();  // the last row's sums are read
#pragma unroll
    for (int e = 0; e < E; e++) s_o[wv][E * lane + e] = o[e];
    if (lane == 0) s_ml[wv] = float2{m, l};
    __syncthreads();
    const int c = threadIdx.x;
    if (c >= D) return;
    m = s_ml[0].x;
#pragma unroll
    for (int w = 1; w < JW; w++) m = fmaxf(m, s_ml[w].x);
    float x = 0.0f;
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < JW; w++) {
        const float f = __builtin_amdgcn_exp2f(s_ml[w].x - m);
        l += s_ml[w].y * f;
        x += s_o[w][c] * f;
    }
    const int tok = a.by_rep.div(r), hq = it.head * a.n_rep + r - tok * a.n_rep;
    x *= visible(a, it, r) > 0 ? 1.0f / l : 0.0f;
    if (a.r.gate)
        x *= sigmoid(((const T*)a.r.gate)[(it.row0 + tok) * a.r.gate_token + hq * a.r.gate_head + c]);
    ((T*)a.r.out)[(it.row0 + tok) * a.r.out_token + hq * a.r.out_head + c] = (T)x;
}

// ------------------------------------------------------------ many rows
typedef __attribute__((address_space(3))) char lds_char;
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return (uint32_t)(uintptr_t)(lds_char*)p;
}
// 16 bytes a lane from g into LDS at to + 16 lane, past the registers.  (Not the
// builtin: behind it the compiler waits for the load before every LDS read.)
__device__ __forceinline__ void load_lds16(const void* g, uint32_t to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g),
                 "s"(__builtin_amdgcn_readfirstlane(to))
                 : "memory");
}
// The same from a uniform address and a lane's bytes.
__device__ __forceinline__ void load_lds16(const void* g, uint32_t bytes, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(bytes), "s"(g),
                 "s"(__builtin_amdgcn_readfirstlane(to))
                 : "memory");
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// Four keys' values of a lane's dim: each 16 lanes read a 4 x 16 block whose
// row j lies at lanes 4 j .. 4 j + 3, and lane i gets its column i.
__device__ __forceinline__ u2 read_tr(const char* p) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                      (__attribute__((address_space(3))) s4*)p));
}

constexpr int TAB = 1024;  // pages whose byte offsets are in LDS (-1: not a page)

// The lane, without a register that holds it until then.
__device__ __forceinline__ int lane_again() {
    int l;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
    return l;
}

// Row r of the item: its output, times the gate, four dims from dim on.
template <typename T>
__device__ __forceinline__ void store_row4(const AttnArgs& a, const Item& it, int r, int dim, f4 o) {
    const int tok = a.by_rep.div(r), hq = it.head * a.n_rep + r - tok * a.n_rep;
    if (a.r.gate) {
        const u2e g = *reinterpret_cast<const u2e*>((const T*)a.r.gate + (it.row0 + tok) * a.r.gate_token +
                                                    hq * a.r.gate_head + dim);
        const typename V<T>::x4 gv = __builtin_bit_cast(typename V<T>::x4, u2{g.x, g.y});
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] *= sigmoid(gv[e]);
    }
    *reinterpret_cast<u2e*>((T*)a.r.out + (it.row0 + tok) * a.r.out_token + hq * a.r.out_head + dim) =
        u2e{pack<T>(o[0], o[1]), pack<T>(o[2], o[3])};
}

// 32 rows a wavefront on 32x32x16 MFMAs, 64 keys and values at a time in one of
// two LDS slots while the next ones are on their way into the other, straight
// from memory.  KG 1: NW wavefronts of 32 NW rows, each taking all 64 keys; KG 2:
// 128 rows, each wavefront 32 of the 64 keys of its rows, the two halves
// joined at the end.  S^T = K Q^T: its result (row = lane % 32, key 8 (e / 4) +
// 4 (lane / 32) + e % 4 in register e) is the B operand of O^T += V^T P^T when
// that product's K index i of step s stands for key 16 s + 8 (i / 4) + 4 (lane /
// 32) + i % 4, which is how V is read, transposed on its way out of LDS.
// 16-byte pieces of a row are permuted (K: piece ^ key, V: piece ^ 4 key) so
// that the lanes of a read meet all banks (no conflict counted).  Bound: the
// matrix cores, beside which a unit's 64 products a wavefront put some 320 vector
// instructions (maximum, exponentials, packing, addresses) and 130 LDS reads:
// busy half of the cycles, at the 2.0 GHz that the power leaves.  A prompt of
// 8,192, 24 / 4 heads of 256 in fp16: 791 to 809 us, 1,020 to 1,043 TFLOP/s (large
// library products: 1,228 to 1,304); 128 tokens after 32,768, KG 2: 803; 32 / 8
// heads of 128, two blocks of 4 wavefronts a CU, a prompt of 8,192: 594 us, 926.
template <typename T, int D, int KG, int NW>
__device__ __forceinline__ void tile_item(const AttnArgs& a, const Part& pt, const Item& it, char* lds) {
    constexpr int NS = D / 16, ND = D / 32;  // K steps of a score, dim tiles
    constexpr int ROW = 2 * D, SLOT = 64 * ROW;  // bytes
    constexpr int CH = D / 8, KPI = 64 / CH;  // pieces a row, keys a load
    constexpr int WK = 64 / NW, NL = WK / KPI;     // keys a wavefront loads, its loads
    constexpr int AHEAD = D == 64 ? 4 : D == 128 ? 6 : 3;
    // Q operands that stay in LDS: a register file holds 128 of O, 64 of Q, 16
    // scores and 16 of operands, and a few too few for what goes with them.
    constexpr int QL = D == 256 ? 2 : 0;
    typedef typename V<T>::x8 x8;
    char* const ks = lds;
    char* const vs = lds + 2 * SLOT;
    long long* const tab = reinterpret_cast<long long*>(lds + 4 * SLOT);
    __shared__ int s_bad;
    __shared__ float2 s_ml[2][4][32];
    const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int ln = lane & 31, hh = lane >> 5;
    const int rg = KG == 1 ? wv : wv & 3, kg = KG == 1 ? 0 : wv >> 2;
    constexpr int BR = 32 * NW / KG;
    const int n_rows = it.n_q * a.n_rep;
    // (a lane of no row is the last row again and stores nothing)
    const int r_in = min(it.qt * BR + rg * 32 + ln, n_rows - 1);
    const int vis = visible(a, it, r_in);
    const int vis_hi = visible(a, it, min(it.qt * BR + BR, n_rows) - 1);
    const int units = (vis_hi + 63) >> 6;
    int u_lo, u_hi;
    split_units(it, units, u_lo, u_hi);
    const float sc2 = score_scale(a.r.scale);
    int w0 = 0;  // first page of the table's window
    auto fill = [&](int u) __attribute__((always_inline)) {
        w0 = a.by_page.div(u * 64);
        const int n = min(TAB, a.by_page.div(vis_hi - 1) + 1 - w0);
        for (int i = wv * 64 + lane_again(); i < n; i += 64 * NW) {
            const int e = a.r.table[(size_t)it.seq * a.r.table_ld + w0 + i];
            const bool bad = (unsigned)e >= (unsigned)a.p.n_pages;
            tab[i] = bad ? -1 : 2 * (e * a.p.page_stride);
            if (bad) s_bad = 1;
        }
    };
    // A unit into a slot: WK keys a wavefront, NL loads of 1 KB of K and of V.  A
    // load takes the address unit 16 cycles, and a wavefront waits where others'
    // are before its own.  So of 8 wavefronts the two of a SIMD, i and i + 4, take
    // turns: i + 4 loads while i has the matrix cores for its scores, and i loads
    // while i + 4 has them (all eight at once, or between their products, left the
    // matrix cores idle half the time: 890 us of a prompt of 8,192 for 840).
    // Where the WK keys lie in one page, as they do in pages of a multiple of WK,
    // an address is a scalar and a lane's constant; else each lane looks its
    // key up.
    const char* const kh = (const char*)a.p.k + 2 * (it.head * a.p.head_stride);
    const char* const vh = (const char*)a.p.v + 2 * (it.head * a.p.head_stride);
    const int last = vis_hi - 1;
    const bool by_group = a.p.page_size % WK == 0 && a.p.token_stride * a.p.page_size < 1 << 28;
    auto stage = [&](int u) __attribute__((always_inline)) {
        const int l = lane_again(), lk = l / CH, p = l % CH;
        const uint32_t to = ((u - u_lo) & 1) * SLOT + wv * NL * 1024;
        auto piece_k = [&](int key) { return (p ^ (D == 64 ? (key >> 1) & 7 : key & 15)) << 4; };
        auto piece_v = [&](int key) { return (p ^ (D == 64 ? (key & 2) << 1 : (key & 3) << 2)) << 4; };
        if (by_group) {
            const int t = min(u * 64 + wv * WK, last & ~(WK - 1)), pg = a.by_page.div(t);
            const int ts2 = 2 * (int)a.p.token_stride;
            const long long at = uniform(max(uniform(tab[pg - w0]), 0ll) + (t - pg * a.p.page_size) * ts2);
            const int most = last - t;
#pragma unroll
            for (int i = 0; i < NL; i++) {
                const int row = i * KPI + lk, key = wv * WK + row, off = min(row, most) * ts2;
                load_lds16(kh + at, off + piece_k(key), lds_addr(ks) + to + i * 1024);
                load_lds16(vh + at, off + piece_v(key), lds_addr(vs) + to + i * 1024);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NL; i++) {
                const int key = wv * WK + i * KPI + lk, t = min(u * 64 + key, last), pg = a.by_page.div(t);
                const long long off = max(tab[pg - w0], 0ll) + 2 * ((t - pg * a.p.page_size) * a.p.token_stride);
                load_lds16(kh + off + piece_k(key), lds_addr(ks) + to + i * 1024);
                load_lds16(vh + off + piece_v(key), lds_addr(vs) + to + i * 1024);
            }
        }
    };
    f16v acc[ND];
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[i][e] = 0.0f;
    float m_ref = M_NONE, l_part = 0.0f;
    // where a lane's operands lie in a slot's 32 keys
    const int k_at = ln * ROW + ((hh ^ (D == 64 ? (ln >> 1) & 7 : ln & 15)) << 4);
    const int vj = (lane >> 2) & 3;
    const int v_at = (4 * hh + vj) * ROW + ((D == 64 ? vj >> 1 : vj) << 6) +
                     (2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) * 16 + (lane & 1) * 8;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    if (u_lo < u_hi) {
        fill(u_lo);
        __syncthreads();
        stage(u_lo);
    }
    x8 qb[NS - QL];
    char* const ql = lds + 4 * SLOT + TAB * (int)sizeof(long long) + wv * (QL * 1024) + lane * 16;
    {
        const uint32_t flip = a.r.scale < 0.0f ? 0x80008000u : 0u;
        const int tok = a.by_rep.div(r_in);
        const T* q = (const T*)a.r.q + (it.row0 + tok) * a.r.q_token +
                     (it.head * a.n_rep + r_in - tok * a.n_rep) * a.r.q_head + 8 * hh;
#pragma unroll
        for (int st = 0; st < NS; st++) {
            const u4e v = *reinterpret_cast<const u4e*>(q + 16 * st);
            const u4 w = {v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip};
            if (st < QL) *reinterpret_cast<u4*>(ql + st * 1024) = w;
            else qb[st - QL] = __builtin_bit_cast(x8, w);
        }
    }
    const int q_at = lds_addr(ql) - lds_addr(lds);
    // unit u is waited for, the next one started
    auto begin = [&](int u) __attribute__((always_inline)) {
        wait_loads();
        __syncthreads();  // u is there, u - 1 is done with
        if (u + 1 < u_hi) {
            if (a.by_page.div(min(u * 64 + 127, vis_hi - 1)) - w0 >= TAB) {
                fill(u);
                __syncthreads();
            }
            if (NW == 4 || wv >= 4) stage(u + 1);
        }
    };
    auto keys = [&](int u, auto masked) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked)::value;
        bool staged = NW == 4 || wv >= 4 || u + 1 >= u_hi;
#pragma unroll 1
        for (int sub = kg; sub < 2; sub += KG) {
            const int key0 = u * 64 + 32 * sub;
            if (MASKED && __ballot(vis > key0) == 0ull) break;  // these keys are no row's
            const int at = ((u - u_lo) & 1) * SLOT + sub * 32 * ROW;
            const char* const kb = ks + at;
            const char* const vb = vs + at;
            const int ka = opaque(k_at), va = opaque(v_at);  // (the permuted places: a xor each)
            // An operand's read is AHEAD products before its own.  (256 dims: the
            // permutation leaves a place's 256s alone, so two reads share a xor.)
            auto step = [](int n) { return D == 256 ? (n >> 1) + (n & 1) * 8 : n; };
            auto tile = [](int n) { return D == 256 ? (n >> 1) + (n & 1) * 4 : n; };
            x8 kf[AHEAD + 1];
            auto read_k = [&](int n) {
                const int st = step(n);
                kf[n % (AHEAD + 1)] = *reinterpret_cast<const x8*>(
                    D == 256 ? kb + (ka ^ ((st & 7) << 5)) + (st >> 3) * 256 : kb + (ka ^ (st << 5)));
            };
            u4 vf[AHEAD + 1];  // dim tile(n / 2), K step n % 2
            auto read_v = [&](int n) {
                const int i = tile(n >> 1);
                const char* const p = (D == 256 ? vb + (va ^ ((i & 3) << 6)) + (i >> 2) * 256 : vb + (va ^ (i << 6))) +
                                      16 * (n & 1) * ROW;
                const u2 lo = read_tr(p), hi = read_tr(p + 8 * ROW);
                vf[n % (AHEAD + 1)] = u4{lo.x, lo.y, hi.x, hi.y};
            };
            f16v sc;
#pragma unroll
            for (int e = 0; e < 16; e++) sc[e] = 0.0f;
#pragma unroll
            for (int n = 0; n < AHEAD; n++) read_k(n);
#pragma unroll
            for (int n = 0; n < NS; n++) {
                const int st = step(n);
                if (n + AHEAD < NS) read_k(n + AHEAD);
                else read_v(n + AHEAD - NS);
                __builtin_amdgcn_sched_barrier(0);
                sc = mfma32(kf[n % (AHEAD + 1)],
                            st < QL ? *reinterpret_cast<const x8*>(lds + q_at + st * 1024) : qb[max(st - QL, 0)], sc);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (!staged) {
                stage(u + 1);
                staged = true;
            }
            bool odd = false;  // values that are no numbers where a row's mask has to hold
            if constexpr (MASKED) {
                if (s_bad) {
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const int t = min(key0 + 8 * (e >> 2) + 4 * hh + (e & 3), vis_hi - 1);
                        if (tab[a.by_page.div(t) - w0] < 0) sc[e] = __builtin_nanf("");
                    }
                }
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (key0 + 8 * (e >> 2) + 4 * hh + (e & 3) >= vis) sc[e] = -INFINITY;
#pragma unroll 4
                for (int i = 0; i < D / 16; i++) {
                    const u4 v = *reinterpret_cast<const u4*>(vb + (i * 64 + lane) * 16);
                    odd = odd || nonfinite_pair<T>(v.x) || nonfinite_pair<T>(v.y) ||
                          nonfinite_pair<T>(v.z) || nonfinite_pair<T>(v.w);
                }
                odd = __ballot(odd) != 0ull;
            }
            float lmax = sc[0];
#pragma unroll
            for (int e = 1; e < 16; e++) lmax = fmaxf(lmax, sc[e]);
            lmax *= sc2;
            if (__ballot(lmax > m_ref + GAP) != 0ull) {
                lmax = fmaxf(lmax, __shfl_xor(lmax, 32, 64));
                const float m_new = fmaxf(m_ref, lmax);
                const float fac = __builtin_amdgcn_exp2f(m_ref - m_new);  // 0 from M_NONE, 1 where it stays
                m_ref = m_new;
                l_part *= fac;
#pragma unroll
                for (int i = 0; i < ND; i++) acc[i] *= fac;
            }
            uint32_t pw[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                pw[e] = pack<T>(__builtin_amdgcn_exp2f(fmaf(sc[2 * e], sc2, -m_ref)),
                                __builtin_amdgcn_exp2f(fmaf(sc[2 * e + 1], sc2, -m_ref)));
                l_part = add_pair<T>(pw[e], l_part);
            }
            x8 pb[2];
#pragma unroll
            for (int sp = 0; sp < 2; sp++)
                pb[sp] = __builtin_bit_cast(x8, u4{pw[4 * sp], pw[4 * sp + 1], pw[4 * sp + 2], pw[4 * sp + 3]});
            if (MASKED && odd) {
                // 0 * inf is no 0: such values join the rows that see them apart
#pragma unroll 1
                for (int k = 0; k < 32; k++) {
                    const int fv = D == 64 ? (k & 2) << 1 : (k & 3) << 2;
                    const bool sees = key0 + k < vis;
#pragma unroll
                    for (int i = 0; i < ND; i++)
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const u2 w = *reinterpret_cast<const u2*>(vb + k * ROW + ((4 * i + q) ^ fv) * 16 + hh * 8);
                            const typename V<T>::x4 v = __builtin_bit_cast(typename V<T>::x4, w);
#pragma unroll
                            for (int c = 0; c < 4; c++) {
                                const float x = (float)v[c];
                                acc[i][4 * q + c] += sees && !(fabsf(x) < INFINITY) ? x : 0.0f;
                            }
                            __builtin_amdgcn_sched_barrier(0);
                        }
                }
            }
#pragma unroll
            for (int n = 0; n < 2 * ND; n++) {
                if (n + AHEAD < 2 * ND) read_v(n + AHEAD);
                __builtin_amdgcn_sched_barrier(0);
                u4 v = vf[n % (AHEAD + 1)];
                if constexpr (MASKED)  // ... and leave the product
                    v = u4{finite_pair<T>(v.x), finite_pair<T>(v.y), finite_pair<T>(v.z), finite_pair<T>(v.w)};
                const int i = tile(n >> 1);
                acc[i] = mfma32(__builtin_bit_cast(x8, v), pb[n & 1], acc[i]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (MASKED && !staged) stage(u + 1);
    };
    if (NW == 8 && wv >= 4) __builtin_amdgcn_s_setprio(1);
    // units that every row sees whole, then the others; all from the first entry
    // outside the cache on
    const int u_mid = min(u_hi, visible(a, it, it.qt * BR) >> 6);
    int u = u_lo;
    bool begun = false;
    for (; u < u_mid; u++) {
        begin(u);
        if ((begun = s_bad != 0)) break;
        keys(u, std::false_type{});
    }
    for (; u < u_hi; u++) {
        if (!begun) begin(u);
        begun = false;
        keys(u, std::true_type{});
    }
    float l_row = l_part + __shfl_xor(l_part, 32, 64);
    constexpr int HD = ND / 2, AREA = 32 * (D / 2) * (int)sizeof(float);
    const int el = lane_again(), eln = el & 31, ehh = el >> 5;
    __syncthreads();  // the slots are free: 32 rows of half the dims for each wavefront
    // Half `half` of the dims: dim 32 i + 8 q + 4 ehh + c of it of row eln in
    // res[i][4 q + c].  (Code that runs once a block costs more to fetch than to
    // run: the halves are a loop, and a row's place is computed by one lane.)
    auto leave_part = [&](const f16v(&res)[HD], int half) __attribute__((always_inline)) {
            const int part = it.part + it.split * a.p.H_kv;
        f4* const x = reinterpret_cast<f4*>(part_acc(a, pt, D, part)) + (rg * ND + half * HD) * (4 * 64) + el;
#pragma unroll
        for (int i = 0; i < HD; i++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                x[(i * 4 + q) * 64] = f4{res[i][4 * q], res[i][4 * q + 1], res[i][4 * q + 2], res[i][4 * q + 3]};
        if (ehh == 0 && half == 0) part_ml(a, pt, D, part)[rg * 32 + eln] = float2{m_ref, l_row};
    };
    // Outputs go through LDS, so that a lane stores 16 bytes next to its
    // neighbours': lane el takes 8-dim group el % GN of row el / GN of RI at once.
    auto leave = [&](const f16v(&res)[HD], int half, char* area) __attribute__((always_inline)) {
        constexpr int CN = D / 8, GN = D / 16, RI = 64 / GN, NR = 32 / RI;
        const int r0 = it.qt * BR + rg * 32, r = min(r0 + eln, n_rows - 1), tok = a.by_rep.div(r);
        const int hq = it.head * a.n_rep + r - tok * a.n_rep;
        const long long to = (it.row0 + tok) * a.r.out_token + hq * a.r.out_head;
        const long long gt = (it.row0 + tok) * a.r.gate_token + hq * a.r.gate_head;
        const int g = el % GN, dim = half * (D / 2) + 8 * g;
        u4 gate[NR];
        if (a.r.gate) {
#pragma unroll
            for (int k = 0; k < NR; k++)
                gate[k] = *reinterpret_cast<const u4e*>((const T*)a.r.gate + __shfl(gt, k * RI + el / GN, 64) + dim);
        }
        const float inv = vis > 0 ? 1.0f / l_row : 0.0f;
        mu::wave_sync();
#pragma unroll
        for (int i = 0; i < HD; i++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                *reinterpret_cast<f4*>(area + eln * (CN * 16) + (((8 * i + 2 * q + ehh) ^ (eln & (CN - 1))) << 4)) =
                    f4{res[i][4 * q], res[i][4 * q + 1], res[i][4 * q + 2], res[i][4 * q + 3]} * inv;
        mu::wave_sync();
#pragma unroll
        for (int k = 0; k < NR; k++) {
            const int row = k * RI + el / GN, s = row & (CN - 1);
            f4 x = *reinterpret_cast<const f4*>(area + row * (CN * 16) + (((2 * g) ^ s) << 4));
            f4 y = *reinterpret_cast<const f4*>(area + row * (CN * 16) + (((2 * g + 1) ^ s) << 4));
            if (a.r.gate) {
                const x8 gv = __builtin_bit_cast(x8, gate[k]);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[e] *= sigmoid(gv[e]);
                    y[e] *= sigmoid(gv[4 + e]);
                }
            }
            const long long o = __shfl(to, row, 64);
            if (r0 + row < n_rows)
                *reinterpret_cast<u4e*>((T*)a.r.out + o + dim) =
                    u4e{pack<T>(x[0], x[1]), pack<T>(x[2], x[3]), pack<T>(y[0], y[1]), pack<T>(y[2], y[3])};
        }
    };
    f16v res[HD];
    if constexpr (KG == 1) {
#pragma unroll
        for (int i = 0; i < HD; i++) res[i] = acc[i];
#pragma unroll 1
        for (int half = 0; half < 2; half++) {
            if (it.n_split == 1) leave(res, half, lds + wv * AREA);
            else leave_part(res, half);
#pragma unroll
            for (int i = 0; i < HD; i++) res[i] = acc[HD + i];
        }
    } else {
        // the two halves of a row's keys: wavefront kg joins and stores half kg of the dims
        auto give = [&](const f16v* from) __attribute__((always_inline)) {
            f4* const x = reinterpret_cast<f4*>(lds + (rg * 2 + kg) * AREA) + el;
#pragma unroll
            for (int i = 0; i < HD; i++)
#pragma unroll
                for (int q = 0; q < 4; q++)
                    x[(i * 4 + q) * 64] = f4{from[i][4 * q], from[i][4 * q + 1], from[i][4 * q + 2], from[i][4 * q + 3]};
        };
        if (kg == 0) {
            give(acc + HD);
#pragma unroll
            for (int i = 0; i < HD; i++) res[i] = acc[i];
        } else {
            give(acc);
#pragma unroll
            for (int i = 0; i < HD; i++) res[i] = acc[HD + i];
        }
        if (ehh == 0) s_ml[kg][rg][eln] = float2{m_ref, l_row};
        __syncthreads();
        const float2 ml = s_ml[1 - kg][rg][eln];
        const float m = fmaxf(m_ref, ml.x);
        const float f1 = __builtin_amdgcn_exp2f(m_ref - m), f2 = __builtin_amdgcn_exp2f(ml.x - m);
        m_ref = m;
        l_row = l_row * f1 + ml.y * f2;
        char* const area = lds + (rg * 2 + 1 - kg) * AREA;
        const f4* const x = reinterpret_cast<const f4*>(area) + el;
#pragma unroll
        for (int i = 0; i < HD; i++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const f4 o = x[(i * 4 + q) * 64];
#pragma unroll
                for (int c = 0; c < 4; c++) res[i][4 * q + c] = res[i][4 * q + c] * f1 + o[c] * f2;
            }
        if (it.n_split == 1) leave(res, kg, area);
        else leave_part(res, kg);
    }
}

// The splits of 32 rows (group rg of the tile), dims 8 piece and on: a wavefront.
template <typename T, int D>
__device__ __forceinline__ void tile_join(const AttnArgs& a, const Part& pt, const Item& it, int rg, int piece) {
    constexpr int ND = D / 32;
    const int i = piece >> 2, q = piece & 3, lane = threadIdx.x & 63, ln = lane & 31, hh = lane >> 5;
    const int r = it.qt * pt.rows + rg * 32 + ln, h_kv = a.p.H_kv;
    if (r >= it.n_q * a.n_rep) return;
    f4 o = {};
    float m = M_NONE, l = 0.0f;
    for (int s0 = 0; s0 < it.n_split; s0 += 8) {
        float2 ml[8];
        f4 v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int s = min(s0 + j, it.n_split - 1);
            ml[j] = part_ml(a, pt, D, it.part + s * h_kv)[rg * 32 + ln];
            v[j] = reinterpret_cast<const f4*>(part_acc(a, pt, D, it.part + s * h_kv))[((rg * ND + i) * 4 + q) * 64 + lane];
        }
        float top = m;
#pragma unroll
        for (int j = 0; j < 8; j++) top = fmaxf(top, ml[j].x);
        const float f0 = __builtin_amdgcn_exp2f(m - top);
        m = top;
        l *= f0;
        o *= f0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (s0 + j >= it.n_split) break;
            const float f = __builtin_amdgcn_exp2f(ml[j].x - m);
            l += ml[j].y * f;
            o += v[j] * f;
        }
    }
    const float inv = visible(a, it, r) > 0 ? 1.0f / l : 0.0f;
    store_row4<T>(a, it, r, 32 * i + 8 * q + 4 * hh, o * inv);
}

// ------------------------------------------------------------ the launches
extern __shared__ __align__(1024) char dyn_lds[];

template <typename T, int D>
__global__ __launch_bounds__(64 * STREAM_WAVES, 2) void attn_stream_kernel(AttnArgs a, Part ps) {
    const Schedule sc = schedule<false>(a, ps, false);
    if ((int)blockIdx.x >= sc.total) return;
    stream_item<T, D, STREAM_WAVES>(a, ps, item_of(a, ps, sc, blockIdx.x, false), dyn_lds);
}

// Tiles of the sequences of many rows, then those of few: a continuous batch's
// decoding sequences run beside its chunks (24 sequences in bf16, 32 / 8 heads of
// 128: 78 us; two launches one after the other and two joins took 105).
template <typename T, int D, int KG, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attn_tile_kernel(AttnArgs a, Part pl, Part ps) {
    const Schedule sl = schedule<true>(a, pl, false);
    const int x = blockIdx.x - sl.total;
    if (x < 0) {
        tile_item<T, D, KG, NW>(a, pl, item_of(a, pl, sl, blockIdx.x, false), dyn_lds);
        return;
    }
    const Schedule sc = schedule<false>(a, ps, false);
    if (x < sc.total) stream_item<T, D, NW>(a, ps, item_of(a, ps, sc, x, false), dyn_lds);
}

// The splits' partial results, in order.  Bound: latency where they are few (4 us
// of one token after 511, 6 after 131,071), else their bytes, which the launch
// before has to have written back (128 rows after 8,192: 31 MB, 10 us).
// row_step: rows of a row tile of 16 that there should be (others follow).
template <typename T, int D, int JW>
__global__ __launch_bounds__(64 * JW) void attn_join_kernel(AttnArgs a, Part pl, Part ps, int row_step) {
    const Schedule sc = schedule<false>(a, ps, true);
    for (int x = blockIdx.x; x < sc.total * row_step; x += gridDim.x) {
        const int k = (int)((uint32_t)x / (uint32_t)row_step);
        const Item it = item_of(a, ps, sc, k, true);
        const int rows = min(16, it.n_q * a.n_rep - it.qt * 16);
        for (int row = x - k * row_step; row < rows; row += row_step) stream_join<T, D, JW>(a, ps, it, row);
    }
    if (pl.slots == 0) return;
    const Schedule sl = schedule<false>(a, pl, true);
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), per = pl.rows / 32 * (D / 8);
    for (int x = blockIdx.x * JW + wv; x < sl.total * per; x += gridDim.x * JW)
        tile_join<T, D>(a, pl, item_of(a, pl, sl, x / per, true), x % per / (D / 8), x % (D / 8));
}

// What a call of these sizes launches.
struct Plan {
    bool tile;  // tiles for sequences of many rows
    Part pl, ps;
    int blocks, waves, kg, joins, join_waves, row_step;
};
size_t part_floats(const Part& pt, int d) { return (size_t)2 * pt.slots * pt.rows * (d + 2); }

// The sizes only choose between the two launches: either serves every sequence.
// Rows a sequence may have up to max_q go by 16 where there are no more, or
// where few keys (max_kv: what the table holds) make little work of them: a tile
// starts and ends in some 20 us, however few its keys.  A prompt of 128, 24 heads
// of 256: 14.5 us by 16, 23.4 in tiles; of 256: 18.4 and 29.9; 128 tokens after
// 1,024, past the bound: 38.3 and 34.5; 16 after 8,192, at it: 38.7 and 39.0.
constexpr double LIGHT = 3.0 * (1 << 28);
Plan plan_of(int n_tok, int n_seq, int H_q, int H_kv, int d, int max_q, double max_kv) {
    const int n_rep = H_q / H_kv, seqs = std::min(n_tok, n_seq);
    const long long rows = (long long)n_tok * n_rep;
    Plan p{};
    p.tile = (long long)max_q * n_rep > SMALL_ROWS && (double)n_tok * H_q * d * max_kv > LIGHT;
    if (p.tile) {
        // 256 dims fill LDS with one block's keys and values: 8 wavefronts on 256
        // rows or, where those tiles would be fewer than the CUs, 128.  Else two
        // blocks of 4 on 128 rows, one of which starts or ends while the other works.
        p.waves = d == 256 ? 8 : 4;
        p.kg = d == 256 && rows / 256 * H_kv < 256 ? 2 : 1;
        const int slots = d == 256 ? 256 : 512;
        // With a block a CU, a share of half the slots: more blocks cost more than
        // they level (3 chunks of 363: 43 us, with 3/4 58).  With two, one that ends
        // early leaves the CU to the other: 3/4 (12 chunks of 41: 43.5 us for 45.3).
        const int room = d == 256 ? slots / 2 : slots / 4 * 3;
        p.pl = Part{32 * p.waves / p.kg, TILE_UNIT, slots, room, SERVE_LARGE, 0};
        p.ps = Part{16, 32 * p.waves, slots, slots / 2, SERVE_SMALL, part_floats(p.pl, d)};
    } else {
        p.waves = STREAM_WAVES;
        p.ps = Part{16, 32 * STREAM_WAVES, STREAM_SLOTS, STREAM_SLOTS / 2, SERVE_ALL, 0};
    }
    // row tiles there may be, and blocks: schedule makes at most `slots` more
    const long long large = p.tile ? (rows / p.pl.rows + seqs) * H_kv : 0;
    const long long small = p.tile ? (long long)seqs * H_kv : (rows / 16 + seqs) * H_kv;
    p.blocks = (int)(large + p.pl.slots + small + p.ps.slots);
    p.row_step = (int)std::min<long long>(16, (long long)max_q * n_rep);
    const long long items = std::min<long long>(p.ps.slots, small) * p.row_step;
    // Few rows may have many splits (one token after 131,071: 105 us with 16
    // wavefronts a row, 110 with 4); many rows fill the chip with 4 (32 sequences: a
    // join of 6 us, with 8 wavefronts 11).
    p.join_waves = !p.tile && items <= 64 ? 16 : 4;
    const long long pieces = std::min<long long>(p.pl.slots, large) * (p.pl.rows / 32) * (d / 8);
    p.joins = (int)std::min<long long>(items + (pieces + p.join_waves - 1) / p.join_waves, 2048);
    return p;
}

// LDS of stream_item.
constexpr int stream_bytes(int waves, int d) { return waves * 16 * (d + 6) * (int)sizeof(float) + 16 * (d + 8) * 2; }

template <typename T, int D>
hipError_t launch(const AttnArgs& a, hipStream_t st) {
    const Plan p = plan_of(a.r.n_tok, a.r.n_seq, a.r.H_q, a.p.H_kv, D, a.r.max_q,
                           (double)a.r.table_ld * a.p.page_size);
    if (p.tile) {
        constexpr int NW = D == 256 ? 8 : 4;
        constexpr int bytes = 4 * 64 * 2 * D + TAB * (int)sizeof(long long) + (D == 256 ? 8 * 2 * 1024 : 0);
        static_assert(bytes >= stream_bytes(NW, D), "the stream's wavefronts join there");
        auto* const k = D < 256 || p.kg == 1 ? attn_tile_kernel<T, D, 1, NW> : attn_tile_kernel<T, D, D == 256 ? 2 : 1, NW>;
        const hipError_t e = ensure_dynamic_lds(reinterpret_cast<const void*>(k), bytes);
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(k, dim3(p.blocks), dim3(64 * NW), bytes, st, a, p.pl, p.ps);
    } else {
        constexpr int bytes = stream_bytes(STREAM_WAVES, D);
        const hipError_t e = ensure_dynamic_lds(reinterpret_cast<const void*>(attn_stream_kernel<T, D>), bytes);
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL((attn_stream_kernel<T, D>), dim3(p.blocks), dim3(64 * STREAM_WAVES), bytes, st, a, p.ps);
    }
    auto* const join = p.join_waves == 16 ? attn_join_kernel<T, D, 16> : attn_join_kernel<T, D, 4>;
    hipLaunchKernelGGL(join, dim3(p.joins), dim3(64 * p.join_waves), 0, st, a, p.pl, p.ps, p.row_step);
    return hipGetLastError();
}

}  // namespace

size_t attn_ws_bytes(int n_tok, int n_seq, int H_q, int H_kv, int head_dim, int max_q) {
    // (tiles' partial results are more than those by 16 rows)
    const Plan p = plan_of(n_tok, n_seq, H_q, H_kv, head_dim, max_q, 1e10);
    return (part_floats(p.pl, head_dim) + part_floats(p.ps, head_dim)) * sizeof(float);
}

hipError_t launch_attn(const AttnArgs& a, hipStream_t st) {
    const bool half = a.p.dtype == KHQ_FP16;
    switch (a.p.head_dim) {
        case 64: return half ? launch<fp16, 64>(a, st) : launch<bf16, 64>(a, st);
        case 128: return half ? launch<fp16, 128>(a, st) : launch<bf16, 128>(a, st);
        default: return half ? launch<fp16, 256>(a, st) : launch<bf16, 256>(a, st);
    }
}

}  // namespace paged
}  // namespace khq
