// Attention of chunks of new tokens over the paged cache on the tensor cores
// (tvb_attention_paged; attn_paged.cu has the formula).
//
// paged_chunk_kernel: one CTA an SM takes its run of tiles (attn_schedule):
// blocks of 128 query rows (new token x query head of the group) of one KV head
// of one sequence against tiles of 128 keys (64, F32).  Products in F32 accuracy:
// over an F16 cache q (times scale log2 e, with a power-of-two exponent a row) and
// p (relative to the maximum less 15, attn_lift) are split into F16 hi + lo planes, K and V are F16 as they are, so every
// product takes two MMAs and the bound is the tensor pipe at twice the algorithmic
// FLOPs; over an F32 cache q, K, p and V are split into three bf16 planes (24 bits
// at any magnitude) and a product takes six MMAs.
//
//   loader warps (a slot of shared memory at a time each): K or V by TMA, a box of
//     rows a lane, page by page (pages that no box of 8 rows divides: by 16-byte
//     cp.async); in V rows behind the last key become zeros.  F32: three warps a
//     slot, loads to registers, planes to the swizzled tile
//   MMA warp: S = Q K^T (K-major operands) into one of two TMEM buffers, then O =
//     P V with P from TMEM and V as the MN-major operand it is in memory (no
//     transpose): PV(j), S(j + 2), PV(j + 1), S(j + 3), ...
//   softmax warps, two groups of 128 threads, thread = row: a group takes every
//     other tile (its own running maximum and sum, p as hi + lo over the S columns
//     in TMEM), so that one group's exponentials run under the other's MMAs.  Both
//     add every tile's O, half of the dimensions each, to registers with the
//     rescaling; a fresh product per tile also keeps the tensor core's truncating
//     sums short (16 MMAs: 3e-7; a sum over 6000 keys in TMEM would lose 1.4e-5).
//     Registers move to these warps (setmaxnreg), and what the roles run between
//     tiles stays in rolled loops: unrolled, instruction fetch took half the time
//   a warp works out the pieces ahead of the others
//
// A masked probability is zero but 0 x inf is not: a loader that finds a
// non-finite value in a V tile that some row does not see whole, or a page that
// does not exist, marks the piece, whose rows are then computed key by key.
#include "attn_paged.h"
#include "prefill.h"
#include "tcgen05.cuh"

namespace tvb {

constexpr int kPcRows = 128, kPcSoft = 8, kPcTeams = 2, kPcMaxSlots = 4;
// What starting and leaving a block costs, in tiles (queries in, first scores, output:
// about 15000 cycles).  4 x 512 tokens over 6000 keys: 3, 5, 8 take 167, 151, 158 us.
constexpr int kPcExtra = 5;

// What depends on the cache's type.
template <typename T>
struct PcType;
template <>
struct PcType<__half> {   // q and p in F16 hi + lo, K and V as they are
    static constexpr int kQPlanes = 2, kPlanes = 1, kKeys = 128, kSlots = 4;
    static constexpr int kTeam = 1;            // warps that load an item together
    static constexpr int kSoftRegs = 200, kAuxRegs = 104, kThreads = 384;
};
template <>
struct PcType<float> {    // everything in three bf16 planes
    static constexpr int kQPlanes = 3, kPlanes = 3, kKeys = 64, kSlots = 2;
    static constexpr int kTeam = 3;
    static constexpr int kSoftRegs = 176, kAuxRegs = 80, kThreads = 512;
};
// Warps 0-7 softmax, then the loaders' teams, the pieces' warp, the MMA's.
template <typename T>
constexpr int pc_piece_warp() {
    return kPcSoft + kPcTeams * PcType<T>::kTeam;
}

// Barriers and flags of a CTA.
struct PcShared {
    uint64_t full[kPcMaxSlots], empty[kPcMaxSlots];
    uint64_t s_full[2], p_full[2], o_full[2], o_read[2];
    uint64_t q_full, drained;
    uint64_t fix[kPcTeams];   // a V tile that its loader looks over
    uint32_t tmem;
    int abort;
    int slow, slow_done;        // warps that compute rows key by key now; how many have done so
    int gone[4];                // a warp of the pair gave up
    int poison[8];              // [piece % 8] = piece + 1: marked
    float f[128];               // q scale log2 e = (hi + lo) f; NaN where it is not finite
    float m[4][128];            // what a tile's p refer to, a row
    AttnRun run;
    uint64_t piece_full[4], piece_empty[4];
    AttnPiece piece[4];         // the pieces to come; tiles 0: no more
    float sum[2][2][128];       // a row's sum and maximum in each group, at the end of a piece
};

template <typename T, int HD>
struct PcSmem {
    using Ty = PcType<T>;
    static constexpr int kQAtom = kPcRows * 128, kAtom = Ty::kKeys * 128;       // rows x 64 dims of 16 bits
    static constexpr int kQPlane = kQAtom * (HD / 64), kPlane = kAtom * (HD / 64);
    static constexpr int kQ = 0;
    static constexpr int kSlots = Ty::kQPlanes * kQPlane;
    static constexpr int kSlot = Ty::kPlanes * kPlane;                          // a tile of K or V
    static constexpr int kShared = kSlots + Ty::kSlots * kSlot;
    static constexpr int kSched = kShared + (int)((sizeof(PcShared) + 127) / 128 * 128);
    static constexpr int kBytes = kSched + (int)sizeof(AttnSchedule) + 1024;   // alignment
};

// Shared-memory descriptor of an MN-major operand in 128-byte-swizzled atoms of
// 64 (MN) x 8 (K): atoms `lbo` bytes apart along MN, 1024 along K.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr, uint32_t lbo) {
    uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(lbo >> 4) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1u << 46;
    d |= (uint64_t)2u << 61;
    return d;
}

// A from TMEM (two F16 a column), B from shared memory.
__device__ __forceinline__ void tc_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two F32 operations an instruction.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}

// (x, y) as three packed bf16 planes, each the rounded rest of the one before: 24
// bits, at any magnitude.
__device__ __forceinline__ void bf16_planes(float x, float y, uint32_t* p0, uint32_t* p1, uint32_t* p2) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(*p0) : "f"(y), "f"(x));
    x -= __uint_as_float(*p0 << 16);
    y -= __uint_as_float(*p0 & 0xffff0000u);
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(*p1) : "f"(y), "f"(x));
    x -= __uint_as_float(*p1 << 16);
    y -= __uint_as_float(*p1 & 0xffff0000u);
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(*p2) : "f"(y), "f"(x));
}

// K and V pools as [page][row][head][dim], boxes of `box` rows of one head and 64
// dimensions; box 0: no maps (cp.async).
struct PcMaps {
    CUtensorMap k, v;
};

__device__ __forceinline__ void pc_cp_async16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

// Whole softmax warp, F16: rows key by key.  All rows of a marked piece (f null), shared by
// the warps; else, of the sixteen rows that this warp stored, those that are not finite
// in `stored` though their query is (f, PcShared).
template <int HD>
__device__ __noinline__ void pc_rows_slow(const PagedAttnArgs& a, const AttnPiece& p, int warp, const float* f, const float* stored) {
    const int first = f ? (warp & 3) * 32 + (warp >> 2) * 16 : warp, last = f ? min(first + 16, p.rows) : p.rows;
#pragma unroll 1
    for (int k = first; k < last; k += f ? 1 : kPcSoft) {
        bool odd = !f;
        if (f && f[k] > 0.f)
            for (int d = threadIdx.x & 31; d < HD; d += 32) odd |= !(fabsf(stored[k * HD + d]) < INFINITY);
        if (__any_sync(0xffffffffu, odd)) attn_row_slow<__half, kPcRows, HD>(a, p, k);
    }
}

// One warp, when a wait gave up: every row of the CTA's run is NaN.
template <typename T, int HD>
__device__ __noinline__ void pc_give_up(const PagedAttnArgs& a, const AttnSchedule& sched, const AttnRun& run, AttnPiece* piece,
                                        int align) {
    constexpr int ND = HD / 32;
    float o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = NAN;
    auto rows = [&](const AttnPiece& p) {
        for (int r = 0; r < p.rows; ++r) attn_row_store<kPcRows, HD, ND>(a, p, r, NAN, -INFINITY, o);
    };
    if (!a.balanced) {
        rows(*piece);   // the only one
        return;
    }
    bool begun = false;
    for (int64_t at = run.u; (at = attn_next<kPcRows, PcType<T>::kKeys, kPcExtra>(a, sched, run, at, align, piece)) != 0;) {
        rows(*piece);
        if (piece->slot == 1) {
            begun = true;
            if ((threadIdx.x & 31) == 0) attn_header(a, piece);
        }
        __syncwarp();
    }
    if (!begun && (threadIdx.x & 31) == 0) attn_header(a, nullptr);
}

template <typename T, int HD>
__global__ void __launch_bounds__(PcType<T>::kThreads, 1)
paged_chunk_kernel(const __grid_constant__ PcMaps maps, const __grid_constant__ PagedAttnArgs a, int box) {
    using Ty = PcType<T>;
    using Sm = PcSmem<T, HD>;
    constexpr bool kF32 = sizeof(T) == 4;
    constexpr int kPcKeys = Ty::kKeys, kPcSlots = Ty::kSlots, kPcThreads = Ty::kThreads;
    constexpr int kPcPieceWarp = pc_piece_warp<T>(), kPcMmaWarp = kPcPieceWarp + 1;
    static_assert(kPcThreads == 32 * (kPcMmaWarp + 1), "warps");
    // TMEM: two buffers of a tile's scores and, in their place, probabilities (8 columns a plane and 16 keys); two of O
    constexpr int kPStep = 8 * Ty::kQPlanes, kSBuf = kF32 ? kPcKeys / 16 * kPStep : kPcKeys, kO = 2 * kSBuf;
    static_assert(kO + 2 * HD <= 512 && kSBuf >= kPcKeys && kSBuf >= kPcKeys / 16 * kPStep, "TMEM");
    extern __shared__ unsigned char pc_smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t raw = smem_u32(pc_smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char* smem = pc_smem_raw + (base - raw);
    PcShared& sh = *reinterpret_cast<PcShared*>(smem + Sm::kShared);
    AttnSchedule& sched = *reinterpret_cast<AttnSchedule*>(smem + Sm::kSched);
    const int align = box ? box : 1;

    // the CTA's pieces: a run of tiles, or the one block of an unbalanced grid
    AttnPiece only;
    bool any = true;
    if (a.balanced) {
        const AttnRun run = attn_run(a, attn_schedule<kPcRows, kPcKeys, kPcExtra, kPcThreads>(a, sched, align));
        pdl_launch_dependents();
        any = run.u < run.end;
        if (threadIdx.x == 0) sh.run = run;
    } else {
        any = attn_block<kPcRows, kPcKeys, kPcThreads>(a, align, &only);
    }
    if (!any) {
        if (a.balanced && threadIdx.x == 0) attn_header(a, nullptr);
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < kPcSlots; ++i) {
            mbar_init(sh.full + i, Ty::kTeam);
            mbar_init(sh.empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(sh.s_full + i, 1);
            mbar_init(sh.p_full + i, kPcSoft / 2);
            mbar_init(sh.o_full + i, 1);
            mbar_init(sh.o_read + i, kPcSoft);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(sh.piece_full + i, 1);
            mbar_init(sh.piece_empty + i, kPcSoft + kPcTeams * Ty::kTeam + 1);
        }
        mbar_init(&sh.q_full, kPcSoft);
        mbar_init(&sh.drained, 1);
        for (int i = 0; i < kPcTeams; ++i) mbar_init(sh.fix + i, 1);
        sh.abort = 0;
        sh.slow = sh.slow_done = 0;
        for (int i = 0; i < 4; ++i) sh.gone[i] = 0;
        for (int i = 0; i < 8; ++i) sh.poison[i] = 0;
        fence_barrier_init();
    }
    if (warp == kPcMmaWarp) tmem_alloc(&sh.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    volatile int* abort_flag = &sh.abort;
    volatile int *slow = &sh.slow, *slow_done = &sh.slow_done;
    auto fail = [&]() {
        *abort_flag = 1;
        if (a.status) atomicOr(a.status, TVB_DEV_TIMEOUT);
    };
    // bounded wait; rows computed key by key may take longer than its limit
    auto landed = [&](uint64_t* bar, int phase) -> bool {
        if (mbar_try_wait(bar, (uint32_t)(phase & 1))) return true;
        int seen = *slow_done;
        while (!mbar_wait_bounded(bar, (uint32_t)(phase & 1))) {
            const int done = *slow_done;
            if (*abort_flag || (done == seen && !*slow)) return false;
            seen = done;
        }
        return true;
    };

    // whole warp: piece i is in sh.piece[i % 4], until done(i)
    auto next = [&](int i) -> bool {
        const bool in = landed(sh.piece_full + (i & 3), i >> 2);
        return __all_sync(0xffffffffu, in) && sh.piece[i & 3].tiles != 0;
    };
    auto done = [&](int i) {
        __syncwarp();
        if (lane == 0) mbar_arrive(sh.piece_empty + (i & 3));
    };

    // registers to the softmax warps: 128 x (200 + 200 + 104) = 384 x 168, 256 x (176 + 80) = 512 x 128, what the CTA was
    // launched with
    static_assert(256 * Ty::kSoftRegs + (kPcThreads - 256) * Ty::kAuxRegs <= kPcThreads * (kF32 ? 128 : 168), "registers");
    if (warp >= kPcSoft) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Ty::kAuxRegs));
    if (warp < kPcPieceWarp) {
        // ---- loaders ---------------------------------------------------------------
        const int w = (warp - kPcSoft) / Ty::kTeam;   // team
        constexpr int kLanes = HD / 8;          // 16-byte chunks, lanes a row (cp.async)
        constexpr int kPass = 32 / kLanes;      // rows a warp instruction
        const int c = lane % kLanes;
        int fixes = 0;
        int issued = -1;   // last item whose boxes were requested on `full`
        if (box && w == 0 && lane == 0) {
            prefetch_tmap(&maps.k);
            prefetch_tmap(&maps.v);
        }
        bool ok = true;
        int item0 = 0;   // items of earlier pieces: K0, K1, then V(j), K(j + 2) for every tile j
        for (int pi = 0; ok && next(pi); ++pi) {
            const AttnPiece& p = sh.piece[pi & 3];
            const int nt = p.tiles, nitems = 2 * nt;
            const int* table = a.s.table + (size_t)p.b * a.s.table_ld;
            const int p_first = p.pos0 + (int)a.gdiv.div((uint32_t)p.row);
            const int p_last = p.pos0 + (int)a.gdiv.div((uint32_t)(p.row + p.rows - 1));
            if constexpr (kF32) {
                // this warp's rows of the tile, every third, kBatch row loads (pairs of rows, HD 64) at a time into two sets
                // of registers in turn, so that one is always under way: the next item's first too, before its slot is
                // free, and its rows' pages, whose L2 prefetch makes up for the few bytes in registers.  More at a time is
                // more code: 6 take 114 us where 3 take 110 (six chunks of up to 300 tokens, window 1024).  Values that
                // are not finite have no planes: their piece goes key by key
                constexpr int kRowLanes = HD / 4, kPer = 32 / kRowLanes, kMine = (kPcKeys + Ty::kTeam - 1) / Ty::kTeam;
                constexpr int kBatch = 3, kBatches = (kMine + kBatch * kPer - 1) / (kBatch * kPer);
                static_assert(kBatches % 2 == 0 && kMine <= 32, "two sets of registers; a lane a row");
                const int first = (warp - kPcSoft) % Ty::kTeam, sub = lane / kRowLanes, d = lane % kRowLanes * 4;
                const int64_t head = (int64_t)p.kvh * a.kv.head_stride + d * 4;
                bool bad = false, odd = false;
                auto is_key = [&](int i) { return i != nitems - 1 && (i == 0 || (i & 1)); };
                auto offsets = [&](int i) -> int64_t {   // of row first + lane * kTeam of item i
                    const int tile = i == 0 ? 0 : is_key(i) ? (i + 1) >> 1 : i == nitems - 1 ? nt - 1 : (i >> 1) - 1;
                    const int my = first + lane * Ty::kTeam, t = p.k0 + tile * kPcKeys + my;
                    if (lane >= kMine || my >= kPcKeys || t >= p.k1) return -1;
                    const int64_t off = paged_offset(a.kv, table, t);
                    bad |= off < 0;
                    if (off >= 0)
                        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"((is_key(i) ? a.kv.k : a.kv.v) + (int64_t)p.kvh * a.kv.head_stride + off), "n"(HD * 4) : "memory");
                    return off;
                };
                auto load = [&](int i, int64_t off, int b, float4 (&x)[kBatch]) {
                    const unsigned char* src = (is_key(i) ? a.kv.k : a.kv.v) + head;
#pragma unroll
                    for (int e = 0; e < kBatch; ++e) {
                        const int64_t o = __shfl_sync(0xffffffffu, off, min((b * kBatch + e) * kPer + sub, 31));
                        x[e] = o >= 0 ? *reinterpret_cast<const float4*>(src + o) : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                };
                auto put = [&](unsigned char* dst, int b, const float4 (&x)[kBatch]) {
#pragma unroll
                    for (int e = 0; e < kBatch; ++e) {
                        const int row = first + ((b * kBatch + e) * kPer + sub) * Ty::kTeam;
                        uint2 u[3];
                        bf16_planes(x[e].x, x[e].y, &u[0].x, &u[1].x, &u[2].x);
                        bf16_planes(x[e].z, x[e].w, &u[0].y, &u[1].y, &u[2].y);
                        const float big = fmaxf(fmaxf(fabsf(x[e].x), fabsf(x[e].y)), fmaxf(fabsf(x[e].z), fabsf(x[e].w)));
                        const float all = x[e].x + x[e].y + x[e].z + x[e].w;
                        odd |= !(big < 3.3e38f) || all != all;
                        if (row < kPcKeys) {
#pragma unroll
                            for (int pl = 0; pl < 3; ++pl)
                                *reinterpret_cast<uint2*>(dst + pl * Sm::kPlane + sw128_offset(row, (d >> 3) & 7)) = u[pl];
                        }
                    }
                };
                float4 x[kBatch], y[kBatch];
                int i = (w - item0) & (kPcTeams - 1);
                int64_t off = -1;
                if (i < nitems) {
                    off = offsets(i);
                    load(i, off, 0, x);
                }
#pragma unroll 1
                for (; i < nitems; i += kPcTeams) {
                    const int gi = item0 + i, sl = gi % kPcSlots;
                    const int64_t off2 = i + kPcTeams < nitems ? offsets(i + kPcTeams) : -1;
                    const bool free_slot = landed(sh.empty + sl, gi / kPcSlots + 1);
                    if (__any_sync(0xffffffffu, !free_slot || *abort_flag)) {
                        fail();
                        ok = false;
                        break;
                    }
                    unsigned char* dst = smem + Sm::kSlots + sl * Sm::kSlot + (d >> 6) * Sm::kAtom + (d & 4) * 2;
#pragma unroll 1
                    for (int b = 0; b < kBatches; b += 2) {
                        load(i, off, b + 1, y);
                        put(dst, b, x);
                        if (b + 2 < kBatches) load(i, off, b + 2, x);
                        put(dst, b + 1, y);
                    }
                    if (bad || odd) *reinterpret_cast<volatile int*>(&sh.poison[pi & 7]) = pi + 1;
                    if (bad) report_bad(a.status);
                    fence_proxy_async_smem_cta();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(sh.full + sl);
                    off = off2;
                    if (i + kPcTeams < nitems) load(i + kPcTeams, off, 0, x);
                }
            } else
            for (int i = 0; i < nitems; ++i) {
                const int gi = item0 + i;
                if (gi % kPcTeams != w) continue;
                const int sl = gi % kPcSlots;
                const uint32_t slot = base + Sm::kSlots + sl * Sm::kSlot;
                const bool is_k = i != nitems - 1 && (i == 0 || (i & 1));
                const int tile = i == 0 ? 0 : is_k ? (i + 1) >> 1 : i == nitems - 1 ? nt - 1 : (i >> 1) - 1;
                const bool free_slot = landed(sh.empty + sl, gi / kPcSlots + 1);
                if (__any_sync(0xffffffffu, !free_slot || *abort_flag)) {
                    fail();
                    ok = false;
                    break;
                }
                const int t0 = p.k0 + tile * kPcKeys, t1 = min(t0 + kPcKeys, p.k1);
                // V rows that some query row does not see must be finite, those behind the last key zero
                const bool look = !is_k && (t1 - t0 < kPcKeys || t1 - 1 > p_first || t0 < p.first ||
                                            (a.window && t0 <= p_last - a.window));
                bool bad = false;
                if (box) {
                    // one box a lane: `box` rows x 64 dimensions
                    const int per = kPcKeys / box, n = per * (HD / 64), row = (lane % per) * box, at = lane / per;
                    int page = -1, in = 0;
                    if (lane < n && t0 + row < p.k1) {
                        const uint32_t t = (uint32_t)(t0 + row), pg = a.kv.page.div(t);
                        in = (int)(t - pg * a.kv.page.d);
                        page = __ldg(table + pg);
                        if ((unsigned)page >= (unsigned)a.kv.n_pages) {
                            page = -1;
                            bad = true;
                        }
                    }
                    const unsigned go = __ballot_sync(0xffffffffu, page >= 0);
                    uint64_t* bar = look ? sh.fix + w : sh.full + sl;
                    if (bad) {
                        *reinterpret_cast<volatile int*>(&sh.poison[pi & 7]) = pi + 1;
                        report_bad(a.status);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_expect_tx(bar, (uint32_t)(__popc(go) * box * 128));
                    __syncwarp();
                    if (page >= 0)
                        tma_load_4d(slot + at * Sm::kAtom + row * 128, is_k ? &maps.k : &maps.v, at * 64, p.kvh, in, page, bar);
                    if (!look) {
                        issued = gi;
                        continue;
                    }
                    const bool in_time = mbar_wait_bounded(bar, (uint32_t)(fixes++ & 1));
                    if (__any_sync(0xffffffffu, !in_time)) {
                        fail();
                        ok = false;
                        break;
                    }
                } else {
                    const unsigned char* src = (is_k ? a.kv.k : a.kv.v) + (int64_t)p.kvh * a.kv.head_stride + c * 16;
#pragma unroll 1
                    for (int r0 = 0; r0 < kPcKeys; r0 += 32) {
                        int64_t off = -1;
                        if (t0 + r0 + lane < p.k1) {
                            off = paged_offset(a.kv, table, t0 + r0 + lane);
                            bad |= off < 0;
                        }
#pragma unroll 4
                        for (int r = 0; r < 32; r += kPass) {
                            const int64_t o = __shfl_sync(0xffffffffu, off, r + lane / kLanes);
                            const int row = r0 + r + lane / kLanes;
                            pc_cp_async16(slot + (c >> 3) * Sm::kAtom + sw128_offset(row, c & 7), src + (o >= 0 ? o : 0), o >= 0);
                        }
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    asm volatile("cp.async.wait_group 0;" ::: "memory");
                    if (bad) {
                        *reinterpret_cast<volatile int*>(&sh.poison[pi & 7]) = pi + 1;
                        report_bad(a.status);
                    }
                }
                if (look) {
                    __syncwarp();
                    uint32_t nonfinite = 0;
                    for (int j = lane; j < Sm::kPlane / 16; j += 32) {
                        const int key = (j * 16 % Sm::kAtom) / 128;
                        uint4* at = reinterpret_cast<uint4*>(smem + Sm::kSlots + sl * Sm::kSlot + j * 16);
                        if (t0 + key >= p.k1) {
                            *at = make_uint4(0u, 0u, 0u, 0u);
                        } else {
                            const uint4 v = *at;
                            const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                nonfinite |= (uint32_t)((u[e] & 0x7C00u) == 0x7C00u) | (uint32_t)((u[e] & 0x7C000000u) == 0x7C000000u);
                        }
                    }
                    if (nonfinite) *reinterpret_cast<volatile int*>(&sh.poison[pi & 7]) = pi + 1;
                }
                fence_proxy_async_smem_cta();
                __syncwarp();
                if (lane == 0) mbar_arrive(sh.full + sl);
            }
            item0 += nitems;
            done(pi);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (box && *abort_flag) {   // no TMA write may outlive the CTA: the last two items cover every slot still in flight
            for (int i = max(w, issued - kPcTeams); i <= issued; i += kPcTeams)
                mbar_wait_bounded(sh.full + i % kPcSlots, (uint32_t)((i / kPcSlots) & 1));
        }
    } else if (warp == kPcPieceWarp) {
        // ---- the pieces, ahead of the others ------------------------------------------
        int64_t at = a.balanced ? sh.run.u : 0;
        for (int pi = 0;; ++pi) {
            if (pi >= 4 && !__all_sync(0xffffffffu, landed(sh.piece_empty + (pi & 3), (pi >> 2) - 1))) break;
            AttnPiece* out = sh.piece + (pi & 3);
            int n = 0;
            if (a.balanced) {
                at = attn_next<kPcRows, kPcKeys, kPcExtra>(a, sched, sh.run, at, align, out);
                n = at != 0;
            } else if (pi == 0) {
                n = only.tiles;
                if (lane == 0) *out = only;
            }
            if (n == 0 && lane == 0) out->tiles = 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(sh.piece_full + (pi & 3));
            if (n == 0) break;
        }
    } else {
        // ---- MMA issuer --------------------------------------------------------------
        constexpr uint32_t kBf16 = kF32 ? (1u << 7) | (1u << 10) : 0u;                   // operands' type
        constexpr uint32_t idesc_s = umma_idesc_f16(kPcRows, kPcKeys) | kBf16;
        constexpr uint32_t idesc_o = umma_idesc_f16(kPcRows, HD) | (1u << 16) | kBf16;   // B is MN-major
        int item = 0, tile = 0;   // over all pieces
        bool ok = true;
        for (int pi = 0; ok && next(pi); ++pi) {
            const AttnPiece& p = sh.piece[pi & 3];
            if (lane == 0) {
                // the products of two operands' planes, the small ones of all steps before the large: the sum is small
                // while most are added.  F32: (0, 2) (1, 1) (2, 0) (0, 1) (1, 0) (0, 0), rolled for the instruction cache
                auto products = [&](auto& product) {
                    if constexpr (kF32) {
#pragma unroll 1
                        for (int i = 0; i < 6; ++i) product((0x010210 >> 4 * i) & 3, (0x001012 >> 4 * i) & 3, i == 0);
                    } else {
                        product(1, 0, true);
                        product(0, 0, false);
                    }
                };
                auto ready = [&]() { return landed(sh.full + item % kPcSlots, item / kPcSlots); };
                auto mma_s = [&](int j) {   // tile j (of all) takes the buffer of P(j - 2)
                    const uint32_t d = tmem + (j & 1) * kSBuf;
                    const uint64_t qd = sw128_desc(base + Sm::kQ), kd = sw128_desc(base + Sm::kSlots + (item % kPcSlots) * Sm::kSlot);
                    tc_fence_after();
                    // plane x of q, plane y of K; addresses in a descriptor count 16 bytes
                    auto product = [&](int x, int y, bool begin) {
#pragma unroll
                        for (int kk = 0; kk < HD / 16; ++kk) {
                            const uint64_t qo = (kk >> 2) * (Sm::kQAtom >> 4) + (kk & 3) * 2 + x * (Sm::kQPlane >> 4);
                            const uint64_t ko = (kk >> 2) * (Sm::kAtom >> 4) + (kk & 3) * 2 + y * (Sm::kPlane >> 4);
                            tc_mma(d, qd + qo, kd + ko, idesc_s, begin && kk == 0 ? 0u : 1u);
                        }
                    };
                    products(product);
                    tc_commit(sh.s_full + (j & 1));
                    tc_commit(sh.empty + item % kPcSlots);
                    ++item;
                };
                const int end = tile + p.tiles;
                ok = landed(&sh.q_full, pi);
                for (int j = tile; ok && j < min(end, tile + 2); ++j) {
                    ok = ready() && (j < 2 || landed(sh.o_full + (j & 1), (j - 2) >> 1));
                    if (ok) mma_s(j);
                }
                for (int j = tile; ok && j < end; ++j) {
                    ok = ready() && (j < 2 || landed(sh.o_read + (j & 1), (j - 2) >> 1)) && landed(sh.p_full + (j & 1), j >> 1);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t vd = sw128_mn_desc(base + Sm::kSlots + (item % kPcSlots) * Sm::kSlot, Sm::kAtom);
                    const uint32_t pt = tmem + (j & 1) * kSBuf, ot = tmem + kO + (j & 1) * HD;
                    auto product = [&](int x, int y, bool begin) {
#pragma unroll
                        for (int kk = 0; kk < kPcKeys / 16; ++kk)
                            tc_mma_ts(ot, pt + kk * kPStep + 8 * x, vd + kk * (2048 >> 4) + y * (Sm::kPlane >> 4), idesc_o,
                                      begin && kk == 0 ? 0u : 1u);
                    };
                    products(product);
                    tc_commit(sh.o_full + (j & 1));
                    tc_commit(sh.empty + item % kPcSlots);
                    ++item;
                    if (j + 2 < end) {
                        ok = ready() && landed(sh.o_full + (j & 1), j >> 1);   // S(j + 2) takes the place of P(j)
                        if (ok) mma_s(j + 2);
                    }
                }
                if (!ok) fail();
            }
            ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
            tile += p.tiles;
            done(pi);
        }
        if (lane == 0) {
            tc_commit(&sh.drained);   // every MMA issued above
            mbar_wait_bounded(&sh.drained, 0u);
        }
        __syncwarp();
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Ty::kSoftRegs));
        // ---- softmax: thread = row; group `half` takes the tiles of its parity, and half of the dimensions ----
        constexpr int kD = HD / 2;   // dimensions of this thread
        const int r = threadIdx.x & 127, half = warp >> 2;
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory"); };
        // one arrival a warp: 32 on one word would take the shared-memory pipe 32 cycles
        auto warp_arrive = [&](uint64_t* bar) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        auto all_landed = [&](uint64_t* bar, int phase) -> bool {
            return __all_sync(0xffffffffu, landed(bar, phase) && !*abort_flag) != 0;
        };
        bool ok = true;
        bool begun = false;   // a cut block that this CTA begins
        int tile = 0;
        for (int pi = 0; ok && next(pi); ++pi) {
            const AttnPiece& p = sh.piece[pi & 3];
            const bool live = r < p.rows;
            const int row = p.row + min(r, p.rows - 1);
            const int t = (int)a.gdiv.div((uint32_t)row);
            const int tok = p.tok0 + t, head = p.kvh * a.group + row - t * a.group;
            const int pos = live ? p.pos0 + t : -1;
            const int p_first = p.pos0 + (int)a.gdiv.div((uint32_t)p.row);
            const int p_last = p.pos0 + (int)a.gdiv.div((uint32_t)(p.row + p.rows - 1));
            {
                // q times scale log2 e as hi + lo planes with a power-of-two factor a row.  A warp takes 16 rows, all
                // requested before the first is used; lane = 4 dimensions (HD 64: two rows a pass).
                constexpr int kPer = 128 / HD, kLoads = 16 / kPer;   // rows a pass, passes
                const int sub = lane / (HD / 4), d = lane % (HD / 4) * 4;
                float4 x[kLoads];
#pragma unroll
                for (int k = 0; k < kLoads; ++k) {
                    const int qr = p.row + min(warp * 16 + k * kPer + sub, p.rows - 1), qt = (int)a.gdiv.div((uint32_t)qr);
                    x[k] = __ldg(reinterpret_cast<const float4*>(a.q + (size_t)(p.tok0 + qt) * a.ldq +
                                                                 (p.kvh * a.group + qr - qt * a.group) * HD + d));
                }
#pragma unroll
                for (int k = 0; k < kLoads; ++k) {
                    const int qr = warp * 16 + k * kPer + sub;
                    const float4 y = make_float4(x[k].x * a.scale2, x[k].y * a.scale2, x[k].z * a.scale2, x[k].w * a.scale2);
                    int e = 0;
                    uint32_t mx = 0;
                    unsigned char* dst = smem + Sm::kQ + (d >> 6) * Sm::kQAtom + sw128_offset(qr, (d >> 3) & 7) + (d & 4) * 2;
                    if constexpr (kF32) {
                        uint2 u[3];
                        bf16_planes(y.x, y.y, &u[0].x, &u[1].x, &u[2].x);
                        bf16_planes(y.z, y.w, &u[0].y, &u[1].y, &u[2].y);
#pragma unroll
                        for (int pl = 0; pl < 3; ++pl) *reinterpret_cast<uint2*>(dst + pl * Sm::kQPlane) = u[pl];
                    } else {
                        // the largest magnitude by its bits, infinities and NaN apart
                        mx = max(max(__float_as_uint(fabsf(y.x)), __float_as_uint(fabsf(y.y))),
                                 max(__float_as_uint(fabsf(y.z)), __float_as_uint(fabsf(y.w))));
                        if constexpr (HD == 128) {
                            mx = __reduce_max_sync(0xffffffffu, mx);
                        } else {
#pragma unroll
                            for (int o = 8; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                        }
                        // 2^e with the largest / 2^e in [2^13, 2^14): both planes of every value that matters are normal F16
                        if (mx > 0u && mx < 0x7f800000u) e = max(-100, min(114, (int)(mx >> 23) - 127 - 13));
                        const float g = __uint_as_float((uint32_t)(127 - e) << 23);
                        const float v[4] = {y.x * g, y.y * g, y.z * g, y.w * g};
                        __half2 hi[2], lo[2];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            hi[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                            const float2 h = __half22float2(hi[i]);
                            lo[i] = __floats2half2_rn(v[2 * i] - h.x, v[2 * i + 1] - h.y);
                        }
                        *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(hi);
                        *reinterpret_cast<uint2*>(dst + Sm::kQPlane) = *reinterpret_cast<const uint2*>(lo);
                    }
                    if (d == 0) sh.f[qr] = !kF32 && mx >= 0x7f800000u ? NAN : __uint_as_float((uint32_t)(127 + e) << 23);
                }
                fence_proxy_async_smem_cta();
                warp_arrive(&sh.q_full);
            }
            uint64_t acc[kD / 2];   // pairs of dimensions
#pragma unroll
            for (int d = 0; d < kD / 2; ++d) acc[d] = 0ull;
            float m = -INFINITY, l = 0.f;   // of this group's tiles
            float mo = -INFINITY;           // what acc refers to
            int added = tile;
            auto add_o = [&](int upto) -> bool {   // acc += O of the tiles before `upto`
                for (; added < upto; ++added) {
                    if (!all_landed(sh.o_full + (added & 1), added >> 1)) return false;
                    tc_fence_after();
                    const float mj = sh.m[added & 3][r], mn = fmaxf(mo, mj);
                    const float c = mo == mn ? 1.f : ex2(mo - mn), e = mj == mn ? 1.f : ex2(mj - mn);
                    mo = mn;
                    const bool plain = __all_sync(0xffffffffu, c == 1.f && e == 1.f);
                    const uint64_t c2 = pack2(c, c), e2 = pack2(e, e);
#pragma unroll
                    for (int h = 0; h < kD / 32; ++h) {
                        uint32_t o[32];
                        tmem_ld32(lanes + kO + (added & 1) * HD + half * kD + h * 32, o);
                        if (!plain) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) acc[16 * h + i] = fma2(acc[16 * h + i], c2, 0ull);
                        }
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            acc[16 * h + i] = fma2(pack2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), e2, acc[16 * h + i]);
                    }
                    tc_fence_before();
                    warp_arrive(sh.o_read + (added & 1));
                }
                return true;
            };
            const int end = tile + p.tiles;
            for (int j = tile + ((tile ^ half) & 1); ok && j < end; j += 2) {
                ok = add_o(j - 1) && all_landed(sh.s_full + (j & 1), j >> 1);
                if (!ok) break;
                const float f = sh.f[r];   // written before the row's scores were
                tc_fence_after();
                const uint32_t sb = lanes + (j & 1) * kSBuf;
                const int t0 = p.k0 + (j - tile) * kPcKeys, t1 = min(t0 + kPcKeys, p.k1);
                const bool edge = t1 - t0 < kPcKeys || t0 < p.first || t1 - 1 > p_first || (a.window && t0 <= p_last - a.window);
                // keys [first, last] of the tile are the row's: bits of the 32 (or 16) from key c on
                const int last = min(t1 - 1, pos) - t0, first = max(p.first, a.window ? pos - a.window + 1 : 0) - t0;
                auto seen = [&](int c) -> uint32_t {
                    const int hi = min(last - c, 31), lo = max(first - c, 0);
                    return hi < lo ? 0u : (0xffffffffu >> (31 - hi)) & (0xffffffffu << lo);
                };
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                float mn, corr, mref;
                auto maximum = [&]() {
                    const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * f;
                    mn = fmaxf(m, kF32 ? mx : attn_lift(mx));   // (bf16 planes have F32's range)
                    corr = m == mn ? 1.f : ex2(m - mn);
                    mref = mn == -INFINITY ? 0.f : mn;
                };
                uint64_t sum[2] = {0ull, 0ull};
                // loops rolled on purpose: what the three roles run between tiles fits the instruction cache
#pragma unroll 1
                for (int c = 0; c < kPcKeys; c += 32) {
                    uint32_t s[32];
                    tmem_ld32(sb + c, s);
                    tmem_wait_ld();
                    if (edge) {
                        const uint32_t mk = seen(c);
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (!(mk & (1u << k))) s[k] = 0xff800000u;   // -infinity
                    }
#pragma unroll
                    for (int k = 0; k < 32; ++k) m4[k & 3] = fmaxf(m4[k & 3], __uint_as_float(s[k]));
                }
                maximum();
                if constexpr (kF32) {
                    // the planes of p take more columns than its scores: from the last keys to the first they only cover
                    // scores that were read
                    const uint64_t m2 = pack2(-mref, -mref);
#pragma unroll 1
                    for (int c = kPcKeys - 16; c >= 0; c -= 16) {   // 16 keys: 8 columns a plane
                        uint32_t zc[16];
                        tmem_ld16(sb + c, zc);
                        tmem_wait_ld();
                        if (edge) {
                            const uint32_t mk = seen(c);
#pragma unroll
                            for (int k = 0; k < 16; ++k)
                                if (!(mk & (1u << k))) zc[k] = 0xff800000u;
                        }
                        uint32_t p0[8], p1[8], p2[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float2 z = unpack2(add2(pack2(__uint_as_float(zc[2 * k]), __uint_as_float(zc[2 * k + 1])), m2));
                            const float x = ex2(z.x), y = ex2(z.y);
                            sum[k & 1] = add2(sum[k & 1], pack2(x, y));
                            bf16_planes(x, y, &p0[k], &p1[k], &p2[k]);
                        }
                        const uint32_t to = sb + c / 16 * kPStep;
                        tmem_st8(to, p0);
                        tmem_st8(to + 8, p1);
                        tmem_st8(to + 16, p2);
                    }
                } else {
                    const uint64_t f2 = pack2(f, f), m2 = pack2(-mref, -mref);
                    const uint64_t minus1 = pack2(-1.f, -1.f);
#pragma unroll 1
                    for (int c = 0; c < kPcKeys; c += 16) {   // 16 keys: 8 columns of hi, 8 of lo, in place of their scores
                        uint32_t zc[16];
                        tmem_ld16(sb + c, zc);
                        tmem_wait_ld();
                        if (edge) {
                            const uint32_t mk = seen(c);
#pragma unroll
                            for (int k = 0; k < 16; ++k)
                                if (!(mk & (1u << k))) zc[k] = 0xff800000u;
                        }
                        uint64_t x[8];
                        uint32_t pl[16];
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            x[k] = fma2(pack2(__uint_as_float(zc[2 * k]), __uint_as_float(zc[2 * k + 1])), f2, m2);
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float2 y = unpack2(x[k]);
                            x[k] = pack2(ex2(y.x), ex2(y.y));
                        }
#pragma unroll
                        for (int k = 0; k < 8; ++k) sum[k & 1] = add2(sum[k & 1], x[k]);
                        // hi: rounded to F16; lo: the rest of that, rounded (of the value's upper 11 bits instead, it
                        // would not make up for what hi loses below 2^-14, always to the same side)
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float2 y = unpack2(x[k]);
                            const __half2 hi = __floats2half2_rn(y.x, y.y);
                            const float2 h = __half22float2(hi), w = unpack2(fma2(pack2(h.x, h.y), minus1, x[k]));
                            const __half2 lo = __floats2half2_rn(w.x, w.y);
                            pl[k] = *reinterpret_cast<const uint32_t*>(&hi);
                            pl[8 + k] = *reinterpret_cast<const uint32_t*>(&lo);
                        }
                        tmem_st16(sb + c, pl);
                    }
                }
                sh.m[j & 3][r] = mn;
                tmem_wait_st();
                tc_fence_before();
                warp_arrive(sh.p_full + (j & 1));
                const float2 both = unpack2(add2(sum[0], sum[1]));
                l = l * corr + (both.x + both.y);
                m = mn;
                ok = add_o(j);
            }
            ok = ok && add_o(end);
            if (!ok) fail();
            // the row's sum from its two groups
            sh.sum[half][0][r] = l;
            sh.sum[half][1][r] = m;
            if (!ok) *reinterpret_cast<volatile int*>(&sh.gone[warp & 3]) = 1;
            pair_sync();
            ok = !*reinterpret_cast<volatile int*>(&sh.gone[warp & 3]);   // both go on or both leave
            l = 0.f;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const float mg = sh.sum[g][1][r];
                l += mg == -INFINITY ? sh.sum[g][0][r] : sh.sum[g][0][r] * ex2(mg - mo);   // (0 or NaN) : rescaled
            }
            m = mo;
            begun = begun || p.slot == 1;
            const bool poisoned = *reinterpret_cast<volatile int*>(&sh.poison[pi & 7]) == pi + 1;
            const int rows0 = (warp & 3) * 32 + half * 16;   // of the sixteen rows that this warp stores
            float z = 0.f;   // NaN where something stored is not finite
            if (ok && !poisoned) {
                // rows through shared memory (the planes of q, all read), so that a warp stores whole rows: chunk c of row
                // r (16 bytes) at c ^ (r % 32), without bank conflicts either way
                const float scale = p.slot >= 0 ? 1.f : attn_inv(l);
                unsigned char* st = smem + Sm::kQ + r * (HD * 4);
#pragma unroll
                for (int c = 0; c < kD / 4; ++c) {
                    const float2 u = unpack2(acc[2 * c]), v = unpack2(acc[2 * c + 1]);
                    *reinterpret_cast<float4*>(st + (((half * (kD / 4) + c) ^ (r & (HD / 4 - 1))) * 16)) =
                        make_float4(u.x * scale, u.y * scale, v.x * scale, v.y * scale);
                }
                if (half == 0 && live) {
                    if (p.slot >= 0) *reinterpret_cast<float2*>(attn_part_sum<kPcRows, HD>(a, blockIdx.x, p.slot, r)) = make_float2(l, m);
                    else if (a.lse) a.lse[(size_t)tok * a.nh + head] = attn_lse(l, m);
                }
                pair_sync();
                constexpr int kPer = 128 / HD;   // rows a pass
                const int sub = lane / (HD / 4), c = lane % (HD / 4);
#pragma unroll 4
                for (int k = 0; k < 16; k += kPer) {
                    const int rr = rows0 + k + sub;
                    if (rr < p.rows) {
                        const float4 v = *reinterpret_cast<const float4*>(smem + Sm::kQ + rr * (HD * 4) + ((c ^ (rr & (HD / 4 - 1))) * 16));
                        const int rt = (int)a.gdiv.div((uint32_t)(p.row + rr));
                        float* to = p.slot >= 0 ? attn_part<kPcRows, HD>(a, blockIdx.x, p.slot, rr)
                                                : a.out + (size_t)(p.tok0 + rt) * a.ldo + (p.kvh * a.group + p.row + rr - rt * a.group) * HD;
                        *reinterpret_cast<float4*>(to + c * 4) = v;
                        if constexpr (!kF32) z = fmaf(v.x, 0.f, fmaf(v.y, 0.f, fmaf(v.z, 0.f, fmaf(v.w, 0.f, z))));
                    }
                }
            }
            // an infinity times a small plane (zero, or of the other sign) is NaN: rows that are not finite though their
            // queries are go key by key as well (F32: their tiles were marked)
            const bool odd = !kF32 && __any_sync(0xffffffffu, z != 0.f);
            if (ok && (poisoned || odd)) {
                if (lane == 0) atomicAdd(&sh.slow, 1);
                if constexpr (kF32) {   // (not by the function: 120 against 110 us for six chunks of up to 300, window 1024)
                    for (int k = warp; k < p.rows; k += kPcSoft) attn_row_slow<T, kPcRows, HD>(a, p, k);
                } else {
                    pc_rows_slow<HD>(a, p, warp, poisoned ? nullptr : sh.f, reinterpret_cast<const float*>(smem + Sm::kQ));
                }
                if (lane == 0) {
                    atomicAdd(&sh.slow_done, 1);
                    atomicSub(&sh.slow, 1);
                }
            }
            if (p.slot == 1 && threadIdx.x == 0) attn_header(a, &p);
            // every row has left (and every sum was read) before the next piece's queries come
            asm volatile("bar.sync 5, %0;" ::"n"(32 * kPcSoft) : "memory");
            volatile int* gone = sh.gone;
            ok = !(gone[0] | gone[1] | gone[2] | gone[3]);   // all go on or all leave: the barrier above counts on it
            tile += p.tiles;
            done(pi);
        }
        if (a.balanced && !begun && threadIdx.x == 0) attn_header(a, nullptr);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kPcMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if (warp == 0 && *abort_flag) pc_give_up<T, HD>(a, sched, sh.run, sh.piece, align);
}

// Pool as a tensor map, or false where its strides do not make one.
static bool pool_map(CUtensorMap* m, const void* p, const PagedKV& kv, int nkv, int hd, int box) {
    const uint64_t dims[4] = {(uint64_t)hd, (uint64_t)nkv, kv.page.d, (uint64_t)kv.n_pages};
    const uint64_t strides[3] = {(uint64_t)(nkv > 1 ? kv.head_stride : kv.row_stride), (uint64_t)kv.row_stride,
                                 (uint64_t)kv.page_stride};
    const uint32_t b[4] = {64u, 1u, (uint32_t)box, 1u};
    return encode_f16_tiled(m, p, 4, dims, strides, b) == TVB_OK;
}

template <typename T, int HD>
static tvb_status launch_chunk(PagedAttnArgs a, cudaStream_t st) {
    using Ty = PcType<T>;
    static int set[kMaxDevices];
    constexpr int smem = PcSmem<T, HD>::kBytes;
    TVB_TRY(allow_smem(reinterpret_cast<const void*>(paged_chunk_kernel<T, HD>), smem, set));
    PcMaps maps = {};
    int box = 0;
    if constexpr (sizeof(T) == 2) {
        // boxes: the largest power of two that divides a page, up to a tile; pages that leave less than 8 rows go by cp.async
        box = 1;
        while (box < Ty::kKeys && a.kv.page.d % (2u * box) == 0) box *= 2;
        if (box < 8 || !pool_map(&maps.k, a.kv.k, a.kv, a.nkv, HD, box) || !pool_map(&maps.v, a.kv.v, a.kv, a.nkv, HD, box)) box = 0;
    }
    // a piece of two tiles still pays for its start (the block's queries) and its partial sums
    a.min_units = 2 + kPcExtra;
    Workspace ws(st);
    dim3 grid;
    if (a.balanced) {
        grid = dim3((unsigned)num_sms());
        TVB_TRY((attn_workspace<kPcRows, HD>(&a, (int)grid.x, &ws)));
    } else {
        grid = dim3((unsigned)(((int64_t)a.s.n_tokens * a.group) / kPcRows + a.s.n_seqs), (unsigned)a.nkv);
    }
    paged_chunk_kernel<T, HD><<<grid, Ty::kThreads, smem, st>>>(maps, a, box);
    TVB_TRY(check_launch("paged_chunk_kernel"));
    return launch_merge<kPcRows, HD>(a, (int)grid.x, st);
}

tvb_status paged_attn_chunk(const PagedAttnArgs& a, int hd, bool f16, cudaStream_t st) {
    if (f16) return hd == 128 ? launch_chunk<__half, 128>(a, st) : launch_chunk<__half, 64>(a, st);
    return hd == 128 ? launch_chunk<float, 128>(a, st) : launch_chunk<float, 64>(a, st);
}

}  // namespace tvb
