// The optimiser's end of a training step over a list of many tensors (include/niw.h):
//
//   niw_grad_norm           N = (sum_t sum_i g_ti^2)^(1/2), or max |g_ti|
//   niw_grad_clip           out = c g,  c = min(1, max_norm / (N + 1e-6))
//   niw_adam_step_tensors   Adam by c g, with decoupled weight decay, without ever writing c g
//
// All are streams of memory -- 2 flops per element for the norm, 3 for clipping, about 18 for Adam -- and move the algorithm's bytes: the
// norm 4 GB of fp32 at 7.1 TB/s and 0.67 GB of bf16 at 6.6, a clip 4 GB at 6.2, an update 9.4 GB at 6.3 (a large fill reaches 6.9, a
// large copy 6.3).  Small lists are bound by two dependent launches of 4 and 6 to 10 us.
//
// The list lies in device memory (the image: one slot per tensor that has elements), so a call is one launch over all tensors, however
// many.  Tensors are cut into chunks, a workgroup handles whole chunks or parts of one, and finds the tensor of its chunk by a search
// that looks at 64 tensors at a time (find_slot).
//
// Sums.  A square of two 24-bit significands has 48 bits: it is exact in double, and so is its exponent for every fp32 value, so the
// sum of squares neither overflows (an fp32 sum does from |g| = 1.8e19) nor loses small gradients.  The fp64 multiply-add per element
// hides behind the memory stream.  The maximum is taken over the bit patterns of |g| as integers, whose order is that of the values
// and puts NaN above infinity: a NaN is never dropped.
#include "niw_common.h"
#include "niw_bf16.h"
#include <math.h>
#include <string.h>
#include <algorithm>
#include <type_traits>
#include <vector>

namespace {

constexpr int kThreads = 256;
constexpr double kClipEps = 1e-6;

// Chunks: 16,384 elements, or 4,096 for lists of less than 16 M elements, whose few large chunks would leave compute units idle (a
// trainer's 1.2 M: clip 17 -> 15 us, of 1000 vectors alike with either).
constexpr int kChunk = 16384, kSmallChunk = 4096;
constexpr long long kSmallList = 1024ll * kChunk;
constexpr int kMaxPieces = 2048;               // (of a kept small list: see build)
// The norm runs on at most kNormBlocks workgroups, four per compute unit, that walk the list with its whole width: 1 GB and up read at
// 7.0 TB/s with 1024, 6.7 with 2048 or 4096, 6.8 with 512 (which costs half-precision lists a quarter: their conversions want more waves).
constexpr int kNormBlocks = 1024;
static_assert(kNormBlocks <= NIW_NORM_WORKSPACE_DOUBLES - 1, "a partial sum per workgroup, behind the total");
// What a clip or an update writes is written by one workgroup per part of a chunk instead: parts of kPart elements in the order of the
// list keep the pages under way at a time few, which the memory rewards (Adam of 335 M bf16 parameters: parts of 1024 elements 1.70 ms,
// of 2048 1.74, of 4096 1.76; the norm's fixed workgroups 2.0 to 2.1; the next part's loads issued before this one's stores 1.75).
// Smaller parts than these reach the rate at which workgroups start.
constexpr int kAdamPart = 1024;
constexpr int kClipPart = 4096, kClipPartWide = 2048;      // (wide: fp32 to fp32, 8 bytes per element; in place 933 us against 963 for 2 GB,
                                                           // but bf16 to fp32 461 against 423 for 335 M)
// Parts in a row per die (part_of): 256 KB of an fp32 stream.  Adam of 335 M bf16 parameters 1.69 -> 1.58 ms (16 parts 1.64, 32 1.59, 128
// 1.68), 2 GB clipped in place 950 -> 927 us; bf16 to fp32 gains nothing (424 to 447 us with any).
constexpr int kAdamStretch = 64, kClipStretchWide = 32;
// The workgroups of a clip or an update join the norm's partial sums themselves as long as they are few (kFoldGrid): saves a launch,
// 3 us of the trainer's 18; with 120,000 workgroups one more launch is cheaper (2 GB in place: 963 us against 973).
constexpr int kFoldGrid = 4096;
// Lists that touch more than the memory-side cache can keep (256 MB, of which other work has a part) go past the caches, non-temporal: Adam
// of 335 M bf16 parameters 1.91 -> 1.74 ms, but of 8 M fp32 ones (128 MB) 35 -> 45 us.  A norm still leaves the last kCache bytes of
// gradients there, which the clip or update behind it reads first: it walks the list backwards.
constexpr int64_t kCache = 192ll << 20;

// ------------------------------------------------------------------------------------------------ the image of a list
enum Form { kFormNorm = 1, kFormClip = 2, kFormAdam = 3 };
struct GradSlot {
    const void* g;
    void* o;
    long long n;
    int first;                                // chunks of the tensors in front of this one
    int types;                                // dtype | out_dtype << 8
};
struct AdamSlot {
    void* p;
    const void* g;
    float* m;
    float* v;
    float* w;                                 // master copy or null
    long long n;
    int first;
    int types;                                // grad_dtype | param_dtype << 8 | group << 16
    long long pad;
};
static_assert(sizeof(GradSlot) == 32 && sizeof(AdamSlot) == 64, "slots are read as 16-byte pieces");

// device side of a table: the slots, then `first` of every slot again as an array of its own for the search
template <class Slot>
struct List {
    const Slot* slots;
    int count, chunks, chunk, parts;
    // the slot of chunk c: its own number in a list whose tensors have a chunk each
    __device__ __forceinline__ int slot_of(int c) const;
};

// The tensor that chunk c belongs to: every lane looks at one of 64 evenly spaced tensors and the vote of the wave narrows the list to
// the stretch behind the last that begins at or before c -- two dependent loads for up to 4096 tensors, where a bisection takes twelve.
__device__ __forceinline__ int find_slot(const int* first, int count, int c) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = count;
    while (n > 1) {
        const int stride = (n + 63) >> 6, at = lane * stride;
        const int v = at < n ? first[lo + at] : 0x7fffffff;
        const int k = __popcll(__ballot(v <= c)) - 1;
        lo += k * stride;
        n = min(stride, n - k * stride);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

template <class Slot>
__device__ __forceinline__ int List<Slot>::slot_of(int c) const {
    return count == chunks ? c : find_slot(reinterpret_cast<const int*>(slots + count), count, c);
}

// A tensor's first chunk begins with its `head`: the elements in front of the first 128-byte boundary of the stream that matters most (the
// one that is written, or the only one that is read).  Everything behind it is walked in whole cache lines of that stream, and of the
// others where they have the same offset, as they have in buckets.
constexpr int kLine = 128;
__host__ __device__ inline int head_of(const void* p, int size, long long n) {
    const int head = (int)((0 - reinterpret_cast<uintptr_t>(p)) & (kLine - 1)) / size;
    return head < n ? head : (int)n;
}
__host__ __device__ inline int size_of(int dtype) { return dtype == NIW_F32 ? 4 : 2; }
__host__ __device__ inline int head_of(const GradSlot& s, bool written) {
    return written ? head_of(s.o, size_of(s.types >> 8), s.n) : head_of(s.g, size_of(s.types & 255), s.n);
}
__host__ __device__ inline int head_of(const AdamSlot& s, bool written) {
    return written ? head_of(s.w ? s.w : s.p, 4, s.n) : head_of(s.g, size_of(s.types & 255), s.n);
}
// chunks of a tensor: enough for either head
template <class Slot>
__host__ __device__ inline long long chunks_of(const Slot& s, int chunk) {
    return (s.n + chunk - 1) / chunk;
}

// f(slot, chunk, head, begin, end) for the chunks of this workgroup (the norm: a fixed number of workgroups)
template <class Slot, class F>
__device__ __forceinline__ void for_chunks(const List<Slot>& list, F f) {
    int lo = 0, hi = 0, head = 0;             // chunks of the slot at hand
    Slot s{};
    for (int c = blockIdx.x; c < list.chunks; c += gridDim.x) {
        if (c < lo || c >= hi) {
            s = list.slots[list.slot_of(c)];
            lo = s.first;
            hi = lo + (int)chunks_of(s, list.chunk);
            head = head_of(s, false);
        }
        // the first chunk holds the head and a whole chunk behind it; the last one ends early or is empty
        const long long begin = c == lo ? 0 : head + (long long)(c - lo) * list.chunk, end = head + (long long)(c - lo + 1) * list.chunk;
        if (begin < s.n) f(s, c, begin == 0 ? head : 0, begin, end < s.n ? end : s.n);
    }
}
// The element of [begin, end) that this thread handles alone, or -1: the `head` ones in front of the aligned stretch (threads 0 ..), and
// those behind the last whole vector of V (threads 128 ..).  One element per thread, so that they wait for memory once together.
template <int V>
__device__ __forceinline__ long long odd_element(int head, long long begin, long long end) {
    static_assert(kLine / 2 <= kThreads / 2 && V <= kThreads / 2, "a thread per element");
    const int tid = threadIdx.x, tail = (int)((end - begin - head) % V);
    if (tid < head) return begin + tid;
    return tid >= kThreads / 2 && tid < kThreads / 2 + tail ? end - tail + (tid - kThreads / 2) : -1;
}
// the part of this workgroup (one workgroup per part), from the list's end backwards; any = false: nothing is left for it
template <class Slot>
struct Part {
    Slot s;
    long long begin, end;
    int head;
    bool any;
};
template <int STRETCH, class Slot>
__device__ __forceinline__ Part<Slot> part_of(const List<Slot>& list) {
    // workgroups go to the eight dies in turn: of every 8 x STRETCH parts each die takes STRETCH that follow each other
    constexpr unsigned kDies = 8, kGroup = kDies * STRETCH;
    unsigned at_grid = blockIdx.x;
    const unsigned group = at_grid / kGroup * kGroup;
    if (STRETCH > 1 && group + kGroup <= gridDim.x) at_grid = group + at_grid % kDies * STRETCH + (at_grid - group) / kDies;
    const int split = list.parts, b = (int)at_grid / split, part = split - 1 - (int)at_grid % split;
    const int c = list.chunks - 1 - b;
    Part<Slot> p{};
    if (c < 0) return p;
    p.s = list.slots[list.slot_of(c)];
    const int head = head_of(p.s, true), step = list.chunk / split;
    const long long at = (long long)(c - p.s.first) * list.chunk + part * step;
    p.head = at == 0 ? head : 0;
    p.begin = at == 0 ? 0 : head + at;
    p.end = head + at + step < p.s.n ? head + at + step : p.s.n;
    p.any = p.begin < p.s.n;
    return p;
}

// ------------------------------------------------------------------------------------------------ elements
// Vectors of four elements (16 bytes of fp32, 8 of the half types) that may begin on any element: the aligned(..) attributes promise the
// compiler no more than that, and gfx950 takes such accesses as one instruction.  (A template argument drops the attribute, so each
// access names its type here: the build treats -Walign-mismatch, which reports the loss, as an error.)
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));

// NT: past the caches (a list that does not fit them anyway leaves them to what does)
template <bool NT>
__device__ __forceinline__ f32x4 get_f4(const float* p) {
    const f32x4_any* const q = reinterpret_cast<const f32x4_any*>(p);
    if constexpr (NT) return __builtin_nontemporal_load(q);
    else return *q;
}
template <bool NT>
__device__ __forceinline__ u32x2 get_u2(const unsigned short* p) {
    const u32x2_any* const q = reinterpret_cast<const u32x2_any*>(p);
    if constexpr (NT) return __builtin_nontemporal_load(q);
    else return *q;
}
template <bool NT>
__device__ __forceinline__ u32x4 get_u4(const char* p) {
    const u32x4_any* const q = reinterpret_cast<const u32x4_any*>(p);
    if constexpr (NT) return __builtin_nontemporal_load(q);
    else return *q;
}
template <bool NT>
__device__ __forceinline__ void put_f4(float* p, f32x4 x) {
    f32x4_any* const q = reinterpret_cast<f32x4_any*>(p);
    if constexpr (NT) __builtin_nontemporal_store(x, q);
    else *q = x;
}
template <bool NT>
__device__ __forceinline__ void put_u2(unsigned short* p, u32x2 x) {
    u32x2_any* const q = reinterpret_cast<u32x2_any*>(p);
    if constexpr (NT) __builtin_nontemporal_store(x, q);
    else *q = x;
}

template <int DT>
__device__ __forceinline__ float widen(unsigned short bits) {
    if constexpr (DT == NIW_BF16) return __builtin_bit_cast(float, (unsigned)bits << 16);
    else return (float)__builtin_bit_cast(_Float16, bits);
}
template <int DT>
__device__ __forceinline__ float load1(const void* p, long long i) {
    if constexpr (DT == NIW_F32) return static_cast<const float*>(p)[i];
    else return widen<DT>(static_cast<const unsigned short*>(p)[i]);
}
template <bool NT, int DT>
__device__ __forceinline__ f32x4 load4(const void* p, long long i) {
    if constexpr (DT == NIW_F32) return get_f4<NT>(static_cast<const float*>(p) + i);
    else {
        const u32x2 w = get_u2<NT>(static_cast<const unsigned short*>(p) + i);
        return f32x4{widen<DT>((unsigned short)w[0]), widen<DT>((unsigned short)(w[0] >> 16)), widen<DT>((unsigned short)w[1]), widen<DT>((unsigned short)(w[1] >> 16))};
    }
}
// rounds to nearest even: bf16 keeps 8 significand bits, fp16 11 (and overflows to infinity above 65504)
template <int DT>
__device__ __forceinline__ unsigned narrow2(float a, float b) {
    if constexpr (DT == NIW_BF16) return niw::pack_bf16(a, b);
    // the fp32 values as they are: without this the compiler folds the multiply-add that made them into v_fma_mixlo_f16, which rounds
    // once to fp16 -- a parameter would then not be its master copy rounded
    asm("" : "+v"(a), "+v"(b));
    return (unsigned)__builtin_bit_cast(unsigned short, (_Float16)a) | (unsigned)__builtin_bit_cast(unsigned short, (_Float16)b) << 16;
}
template <int DT>
__device__ __forceinline__ void store1(void* p, long long i, float x) {
    if constexpr (DT == NIW_F32) static_cast<float*>(p)[i] = x;
    else static_cast<unsigned short*>(p)[i] = (unsigned short)narrow2<DT>(x, 0.f);
}
template <bool NT, int DT>
__device__ __forceinline__ void store4(void* p, long long i, f32x4 x) {
    if constexpr (DT == NIW_F32) put_f4<NT>(static_cast<float*>(p) + i, x);
    else put_u2<NT>(static_cast<unsigned short*>(p) + i, u32x2{narrow2<DT>(x[0], x[1]), narrow2<DT>(x[2], x[3])});
}
// f(std::integral_constant dtype) for the dtype of a descriptor: the branch is the same for a whole workgroup
template <class F>
__device__ __forceinline__ void with_dtype(int dtype, F f) {
    if (dtype == NIW_F32) f(std::integral_constant<int, NIW_F32>{});
    else if (dtype == NIW_BF16) f(std::integral_constant<int, NIW_BF16>{});
    else f(std::integral_constant<int, NIW_F16>{});
}

// ------------------------------------------------------------------------------------------------ reductions
template <int KIND>
__device__ __forceinline__ double join(double a, double b) {
    if constexpr (KIND == NIW_NORM_2) return a + b;
    else return a != a ? a : (b != b ? b : (a > b ? a : b));
}
template <int KIND>
__device__ __forceinline__ double block_total(double x) {
    __shared__ double part[kThreads / 64];
#pragma unroll
    for (int m = 32; m; m >>= 1) x = join<KIND>(x, __shfl_xor(x, m, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = part[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) x = join<KIND>(x, part[w]);
    return x;
}

// what one thread has seen: four running sums (the fp64 units want more than one chain), or the largest bit pattern
template <int KIND>
struct Seen {
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
    unsigned top = 0;
    __device__ __forceinline__ void operator()(int k, float x) {
        if constexpr (KIND == NIW_NORM_2) sum[k & 3] = fma((double)x, (double)x, sum[k & 3]);
        else top = max(top, __builtin_bit_cast(unsigned, x) & 0x7fffffffu);
    }
    __device__ __forceinline__ double total() const {
        if constexpr (KIND == NIW_NORM_2) return (sum[0] + sum[1]) + (sum[2] + sum[3]);
        else return (double)__builtin_bit_cast(float, top);
    }
};
template <int KIND, int DT, bool NT>
__device__ __forceinline__ void see(Seen<KIND>& seen, const void* p, int head, long long begin, long long end) {
    constexpr int V = DT == NIW_F32 ? 4 : 8, U = 4;      // 16 bytes per thread and load, U loads under way
    const int tid = threadIdx.x;
    auto words = [&](long long i) { return get_u4<NT>(static_cast<const char*>(p) + i * (16 / V)); };
    auto take = [&](u32x4 w) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned bits = w[k];          // (a copy: clang's bit_cast of a vector element in place reads element 0)
            if constexpr (DT == NIW_F32) seen(k, __builtin_bit_cast(float, bits));
            else { seen(2 * k, widen<DT>((unsigned short)bits)); seen(2 * k + 1, widen<DT>((unsigned short)(bits >> 16))); }
        }
    };
    const long long odd = odd_element<V>(head, begin, end);
    const float alone = odd >= 0 ? load1<DT>(p, odd) : 0.f;
    long long i = begin + head;
    for (; i + (long long)kThreads * V * U <= end; i += (long long)kThreads * V * U) {
        u32x4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = words(i + (u * kThreads + tid) * V);
#pragma unroll
        for (int u = 0; u < U; ++u) take(w[u]);
    }
    for (i += tid * V; i + V <= end; i += kThreads * V) take(words(i));
    seen(0, alone);
}

template <int KIND>
__device__ __forceinline__ double norm_of(double total) { return KIND == NIW_NORM_2 ? sqrt(total) : total; }

// Partial sums of the norm: kNormBlocks workgroups walk the list side by side, four loads of 16 bytes per thread under way; bound by HBM
// reads (4 GB fp32 556 us), by its own start where the list is small (1.2 M values 4.8 us).
// total, norm: for a launch of one workgroup, whose sum is the total; null otherwise.  Chunks in front of `cached` are read past the caches: what a clip reads again is the end of the list
template <int KIND, class Slot>
__global__ __launch_bounds__(kThreads) void partial_kernel(List<Slot> list, int cached, double* __restrict__ partial, double* __restrict__ total, float* __restrict__ norm) {
    Seen<KIND> seen;
    for_chunks(list, [&](const Slot& s, int c, int head, long long begin, long long end) {
        with_dtype(s.types & 255, [&](auto dt) {
            if (c < cached) see<KIND, decltype(dt)::value, true>(seen, s.g, head, begin, end);
            else see<KIND, decltype(dt)::value, false>(seen, s.g, head, begin, end);
        });
    });
    const double sum = block_total<KIND>(seen.total());
    if (threadIdx.x) return;
    partial[blockIdx.x] = sum;
    if (total) total[0] = sum;
    if (norm) norm[0] = (float)norm_of<KIND>(sum);
}

// the total of n partial sums, in every thread: the same order wherever it is formed
template <int KIND>
__device__ __forceinline__ double total_of(const double* __restrict__ partial, int n) {
    if (n == 1) return partial[0];
    double x = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) x = join<KIND>(x, partial[i]);
    return block_total<KIND>(x);
}
template <int KIND>
__global__ __launch_bounds__(kThreads) void finish_kernel(const double* __restrict__ partial, int n, double* __restrict__ total, float* __restrict__ norm) {
    const double x = n ? total_of<KIND>(partial, n) : 0.0;
    if (threadIdx.x == 0) {
        if (total) total[0] = x;
        if (norm) norm[0] = (float)norm_of<KIND>(x);
    }
}

// what a clip goes by: n_partial sums of the norm's launch (or the one total), joined by every workgroup for itself
struct Clip {
    const double* partial;                    // null: no clip
    float* norm_out;
    double max_norm;
    int n_partial, skip_nonfinite;
};
struct Factor {
    float c;
    bool skip;                                // leave everything as it is
};
template <int KIND>
__device__ __forceinline__ Factor clip_factor(const Clip& clip) {
    if (!clip.partial) return Factor{1.f, false};
    const double norm = norm_of<KIND>(total_of<KIND>(clip.partial, clip.n_partial));
    if (clip.norm_out && blockIdx.x == 0 && threadIdx.x == 0) clip.norm_out[0] = (float)norm;
    Factor f{1.f, clip.skip_nonfinite && !isfinite(norm)};
    if (isinf(clip.max_norm)) return f;
    const double c = clip.max_norm / (norm + kClipEps);
    if (c < 1.0 || c != c) f.c = (float)c;
    return f;
}

// out = c g, one part per workgroup.  The factor comes first: in place with c = 1 nothing is read.  (Loading the part before the factor is
// known gained nothing out of place and cost 3 % in place.)  2 GB in place 647 us behind a norm of 290; 335 M bf16 to fp32 319 behind 108.
template <int KIND, bool NT, int PART>
__global__ __launch_bounds__(kThreads) void clip_kernel(List<GradSlot> list, Clip clip) {
    const float c = clip_factor<KIND>(clip).c;
    const auto part = part_of<PART == kClipPartWide ? kClipStretchWide : 1>(list);
    const GradSlot& s = part.s;
    if (!part.any || (c == 1.f && s.o == s.g)) return;
    with_dtype(s.types & 255, [&](auto gt) {
        with_dtype(s.types >> 8, [&](auto ot) {
            constexpr int G = decltype(gt)::value, O = decltype(ot)::value, U = PART / (kThreads * 4);
            const int tid = threadIdx.x;
            const long long odd = odd_element<4>(part.head, part.begin, part.end);
            if (odd >= 0) store1<O>(s.o, odd, c * load1<G>(s.g, odd));
            long long i = part.begin + part.head;
            for (; i + kThreads * 4 * U <= part.end; i += kThreads * 4 * U) {
                f32x4 x[U];
#pragma unroll
                for (int u = 0; u < U; ++u) x[u] = load4<NT, G>(s.g, i + (u * kThreads + tid) * 4);
#pragma unroll
                for (int u = 0; u < U; ++u) store4<NT, O>(s.o, i + (u * kThreads + tid) * 4, c * x[u]);
            }
            for (i += tid * 4; i + 4 <= part.end; i += kThreads * 4) store4<NT, O>(s.o, i, c * load4<NT, G>(s.g, i));
        });
    });
}

// 1 - decay as the sum of two fp32 numbers.  p (1 - decay) is fma(p, hi, p lo): rounded once, where 1 - decay rounded to fp32 would keep three
// digits of a decay of 1e-5 and none of one below 2^-25, and p - decay p has no value for an infinite p and loses the sign of a zero.
// So that those come out as products too, lo has the sign of hi (hi is rounded towards zero) and is never 0 beside a hi that is not: 2^-100 of p is
// far below its last bit.  One instruction more per element than p - decay p; asking each p for its class instead took 1 % (335 M bf16
// parameters) to 4 % (101 M fp32 with fp16 gradients) of the update.
struct Keep {
    float hi, lo;
};
__host__ __device__ inline Keep keep_of(float decay) {
    const double k = 1.0 - (double)decay;
    float hi = (float)k;
    if (!(k - k == 0.0)) return Keep{hi, hi};                    // (a decay_dev that is not finite)
    if (fabs((double)hi) > fabs(k)) hi = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, hi) - 1u);
    const float lo = (float)(k - (double)hi);
    return Keep{hi, lo == 0.f && hi != 0.f ? copysignf(0x1p-100f, hi) : lo};
}

struct AdamArgs {
    float step_size[NIW_ADAM_MAX_GROUPS], bc2_sqrt[NIW_ADAM_MAX_GROUPS];
    Keep keep[NIW_ADAM_MAX_GROUPS];
    float w1, b2, w2, eps;
    const float* hyper_dev;
    const float* decay_dev;
};

// The update, one part of 1024 elements per workgroup: four elements of every stream per thread, 28 to 30 bytes each, and nothing reused.
// 335 M bf16 parameters with master copies 1483 us, 101 M fp32 with fp16 gradients in unaligned tensors 417 us.
// DECAY: some group of the call decays (groups that do not then have keep = {1, 2^-100}, which changes no bit).
template <int KIND, bool NT, bool DECAY>
__global__ __launch_bounds__(kThreads) void adam_tensors_kernel(List<AdamSlot> list, AdamArgs a, Clip clip) {
    const Factor factor = clip_factor<KIND>(clip);
    const auto part = part_of<kAdamStretch>(list);
    if (!part.any || factor.skip) return;
    const AdamSlot& s = part.s;
    const int k = __builtin_amdgcn_readfirstlane(s.types >> 16), tid = threadIdx.x;
    const float step_size = a.hyper_dev ? a.hyper_dev[2 * k] : a.step_size[k], bc2_sqrt = a.hyper_dev ? a.hyper_dev[2 * k + 1] : a.bc2_sqrt[k];
    Keep keep{};
    if constexpr (DECAY) keep = a.decay_dev ? keep_of(a.decay_dev[k]) : a.keep[k];
    float* const w = s.w ? s.w : static_cast<float*>(s.p);
    with_dtype(s.types & 255, [&](auto gt) {
        with_dtype((s.types >> 8) & 255, [&](auto pt) {
            constexpr int G = decltype(gt)::value, P = decltype(pt)::value;
            auto update = [&](float& p, float g, float& m, float& v) {
                if constexpr (DECAY) p = fmaf(p, keep.hi, niw::mul_rn(p, keep.lo));
                niw::adam_update(p, niw::mul_rn(factor.c, g), m, v, a.w1, a.b2, a.w2, a.eps, step_size, bc2_sqrt);
            };
            const long long odd = odd_element<4>(part.head, part.begin, part.end);
            if (odd >= 0) {
                float p = w[odd], m = s.m[odd], v = s.v[odd];
                update(p, load1<G>(s.g, odd), m, v);
                w[odd] = p; s.m[odd] = m; s.v[odd] = v;
                if constexpr (P != NIW_F32) store1<P>(s.p, odd, p);
            }
            for (long long i = part.begin + part.head + tid * 4; i + 4 <= part.end; i += kThreads * 4) {
                f32x4 p = load4<NT, NIW_F32>(w, i), m = load4<NT, NIW_F32>(s.m, i), v = load4<NT, NIW_F32>(s.v, i);
                const f32x4 g = load4<NT, G>(s.g, i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float pj = p[j], mj = m[j], vj = v[j];
                    update(pj, g[j], mj, vj);
                    p[j] = pj; m[j] = mj; v[j] = vj;
                }
                store4<NT, NIW_F32>(w, i, p);
                store4<NT, NIW_F32>(s.m, i, m);
                store4<NT, NIW_F32>(s.v, i, v);
                if constexpr (P != NIW_F32) store4<NT, P>(s.p, i, p);
            }
        });
    });
}

// a piece of a host image, by value
struct Piece {
    u32x4 d[240];
};
__global__ __launch_bounds__(kThreads) void store_kernel(Piece piece, u32x4* __restrict__ dst, int n) {
    if ((int)threadIdx.x < n) dst[threadIdx.x] = piece.d[threadIdx.x];
}

// ------------------------------------------------------------------------------------------------ host
bool known(int dtype) { return dtype == NIW_F32 || dtype == NIW_BF16 || dtype == NIW_F16; }
bool aligned(const void* p, int size) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(size - 1)) == 0; }
constexpr int64_t kMaxElements = 1ll << 44, kMaxTensors = 1ll << 20;
// A launch counts its threads in 32 bits: fewer than 2^24 workgroups.  (The norm's are few; its chunks are counted in 31 bits.)
constexpr int64_t kMaxGrid = (1ll << 32) / kThreads - 1;
int64_t max_chunks(int form) {
    return form == kFormNorm ? 1ll << 30 : kMaxGrid / (kChunk / (form == kFormClip ? kClipPartWide : kAdamPart));
}
int64_t padded(int64_t bytes) { return (bytes + 15) / 16 * 16; }

// a range of memory that the call writes (or only reads), for the overlap check
struct Range {
    uintptr_t begin, end;
    int64_t tensor;
    bool writes;
};
int check_overlaps(const char* what, std::vector<Range>& r) {
    std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
    // sweep: the furthest end so far of what is read and of what is written
    uintptr_t read_end = 0, write_end = 0;
    int64_t reader = -1, writer = -1;
    for (const Range& x : r) {
        NIW_REQUIRE(x.begin >= write_end, "%s: tensors %lld and %lld overlap", what, (long long)writer, (long long)x.tensor);
        NIW_REQUIRE(!x.writes || x.begin >= read_end, "%s: tensors %lld and %lld overlap", what, (long long)reader, (long long)x.tensor);
        if (x.writes) { if (x.end > write_end) { write_end = x.end; writer = x.tensor; } }
        else if (x.end > read_end) { read_end = x.end; reader = x.tensor; }
    }
    return NIW_OK;
}
void add_range(std::vector<Range>& r, const void* p, int64_t n, int size, int64_t tensor, bool writes) {
    if (n > 0) r.push_back(Range{reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + (uintptr_t)n * size, tensor, writes});
}

int check_grads(const char* what, const niw_grad_tensor* t, int64_t count, bool for_clip) {
    for (int64_t i = 0; i < count; ++i) {
        NIW_REQUIRE(t[i].n >= 0 && t[i].n <= kMaxElements, "%s: tensor %lld has n=%lld", what, (long long)i, (long long)t[i].n);
        NIW_REQUIRE(known(t[i].dtype), "%s: tensor %lld has unknown dtype %d", what, (long long)i, t[i].dtype);
        NIW_REQUIRE(t[i].n == 0 || t[i].grad, "%s: null pointer in tensor %lld", what, (long long)i);
        NIW_REQUIRE(aligned(t[i].grad, size_of(t[i].dtype)), "%s: tensor %lld is not aligned to its elements", what, (long long)i);
        if (!for_clip) continue;
        NIW_REQUIRE(known(t[i].out_dtype), "%s: output %lld has unknown dtype %d", what, (long long)i, t[i].out_dtype);
        NIW_REQUIRE(t[i].n == 0 || t[i].out, "%s: null pointer in output %lld", what, (long long)i);
        NIW_REQUIRE(aligned(t[i].out, size_of(t[i].out_dtype)), "%s: output %lld is not aligned to its elements", what, (long long)i);
        NIW_REQUIRE(t[i].n == 0 || t[i].out != t[i].grad || t[i].out_dtype == t[i].dtype, "%s: tensor %lld in place changes its type", what, (long long)i);
    }
    if (!for_clip) return NIW_OK;
    std::vector<Range> r;
    r.reserve(2 * count);
    for (int64_t i = 0; i < count; ++i) {
        if (t[i].out != t[i].grad) add_range(r, t[i].grad, t[i].n, size_of(t[i].dtype), i, false);
        add_range(r, t[i].out, t[i].n, size_of(t[i].out_dtype), i, true);
    }
    return check_overlaps(what, r);
}

int check_adam(const char* what, const niw_adam_tensor* t, int64_t count, int n_groups) {
    for (int64_t i = 0; i < count; ++i) {
        const niw_adam_tensor& x = t[i];
        NIW_REQUIRE(x.n >= 0 && x.n <= kMaxElements, "%s: tensor %lld has n=%lld", what, (long long)i, (long long)x.n);
        NIW_REQUIRE(known(x.param_dtype) && known(x.grad_dtype), "%s: tensor %lld has unknown dtype %d / %d", what, (long long)i, x.param_dtype, x.grad_dtype);
        NIW_REQUIRE(x.group >= 0 && x.group < n_groups, "%s: tensor %lld is of group %d of %d", what, (long long)i, x.group, n_groups);
        NIW_REQUIRE(x.n == 0 || (x.param && x.grad && x.exp_avg && x.exp_avg_sq), "%s: null pointer in tensor %lld", what, (long long)i);
        NIW_REQUIRE(x.n == 0 || (x.param_dtype == NIW_F32) == (x.master == nullptr), "%s: tensor %lld: a half-precision parameter, and only one, has a master copy", what,
                    (long long)i);
        NIW_REQUIRE(aligned(x.param, size_of(x.param_dtype)) && aligned(x.grad, size_of(x.grad_dtype)) && aligned(x.exp_avg, 4) && aligned(x.exp_avg_sq, 4) && aligned(x.master, 4),
                    "%s: tensor %lld is not aligned to its elements", what, (long long)i);
    }
    std::vector<Range> r;
    r.reserve(5 * count);
    for (int64_t i = 0; i < count; ++i) {
        add_range(r, t[i].param, t[i].n, size_of(t[i].param_dtype), i, true);
        add_range(r, t[i].grad, t[i].n, size_of(t[i].grad_dtype), i, false);
        add_range(r, t[i].exp_avg, t[i].n, 4, i, true);
        add_range(r, t[i].exp_avg_sq, t[i].n, 4, i, true);
        if (t[i].master) add_range(r, t[i].master, t[i].n, 4, i, true);
    }
    return check_overlaps(what, r);
}

void fill(GradSlot& s, const niw_grad_tensor& t) {
    s.g = t.grad; s.o = t.out; s.n = t.n; s.types = t.dtype | t.out_dtype << 8;
}
void fill(AdamSlot& s, const niw_adam_tensor& t) {
    s.p = t.param; s.g = t.grad; s.m = t.exp_avg; s.v = t.exp_avg_sq; s.w = t.master; s.n = t.n; s.pad = 0;
    s.types = t.grad_dtype | t.param_dtype << 8 | t.group << 16;
}

// bytes of gradients, and bytes that a clip or an update of the tensor touches
void count_bytes(const niw_grad_tensor& t, int64_t& read, int64_t& touched) {
    read += t.n * size_of(t.dtype); touched += t.n * (size_of(t.dtype) + (t.out == t.grad ? 0 : size_of(t.out_dtype)));
}
void count_bytes(const niw_adam_tensor& t, int64_t& read, int64_t& touched) {
    read += t.n * size_of(t.grad_dtype); touched += t.n * (12 + size_of(t.grad_dtype) + (t.master ? 2 : 0));
}
int bytes_per_element(const niw_grad_tensor& t) { return size_of(t.dtype) + size_of(t.out_dtype); }
int bytes_per_element(const niw_adam_tensor&) { return 0; }

// the elements [at, at + n) of a slot
void advance(GradSlot& s, long long at, long long n) {
    s.g = static_cast<const char*>(s.g) + at * size_of(s.types & 255);
    s.o = static_cast<char*>(s.o) + at * size_of(s.types >> 8);
    s.n = n;
}
void advance(AdamSlot& s, long long at, long long n) {
    s.p = static_cast<char*>(s.p) + at * size_of((s.types >> 8) & 255);
    s.g = static_cast<const char*>(s.g) + at * size_of(s.types & 255);
    s.m += at; s.v += at;
    if (s.w) s.w += at;
    s.n = n;
}

template <class Slot, class Item>
int build(const char* what, const Item* items, int64_t count, int form, int groups, bool kept, void* image, niw_table* table) {
    long long total = 0, pieces = 0, wide = 0;
    int slots = 0;
    *table = niw_table{};
    for (int64_t i = 0; i < count; ++i) {
        total += items[i].n; slots += items[i].n > 0;
        pieces += items[i].n / (kSmallChunk - kLine) + 1;
        count_bytes(items[i], table->read, table->touched);
        wide += items[i].n * bytes_per_element(items[i]);
    }
    const int chunk = total < kSmallList ? kSmallChunk : kChunk;
    // small lists that are kept: a slot per chunk, so that no workgroup has to search
    const bool cut = kept && chunk == kSmallChunk && pieces <= kMaxPieces;
    std::vector<Slot> list;
    list.reserve(cut ? pieces : slots);
    long long chunks = 0;
    for (int64_t i = 0; i < count; ++i) {
        if (items[i].n == 0) continue;
        Slot whole{};
        fill(whole, items[i]);
        for (long long at = 0, n; at < items[i].n; at += n) {
            n = items[i].n - at;
            if (cut) {
                // (a first piece ends where the written stream begins a line)
                const int head = at == 0 ? head_of(whole, form != kFormNorm) : 0;
                n = std::min<long long>(n, head ? head + chunk - kLine : chunk);
            }
            Slot s = whole;
            advance(s, at, n);
            s.first = (int)chunks;
            list.push_back(s);
            chunks += chunks_of(s, chunk);
            NIW_REQUIRE(chunks <= max_chunks(form), "%s: more than %lld chunks of %d elements", what, (long long)max_chunks(form), chunk);
        }
    }
    slots = (int)list.size();
    table->form = form; table->slots = slots; table->chunks = (int)chunks; table->chunk = chunk; table->groups = groups;
    table->wide = wide >= 8 * total;
    // as many parts as a chunk has on the average
    const int part = form == kFormAdam ? kAdamPart : table->wide ? kClipPartWide : kClipPart;
    table->parts = 1;
    while (table->parts * part < chunk && table->parts * part * chunks < total) table->parts *= 2;
    table->bytes = padded((int64_t)slots * (sizeof(Slot) + sizeof(int)));
    if (!slots) return NIW_OK;
    memset(image, 0, table->bytes);
    memcpy(image, list.data(), slots * sizeof(Slot));
    int* first = reinterpret_cast<int*>(static_cast<Slot*>(image) + slots);
    for (int i = 0; i < slots; ++i) first[i] = list[i].first;
    return NIW_OK;
}

template <class Slot>
List<Slot> list_of(const niw_table& t) {
    return List<Slot>{static_cast<const Slot*>(t.image), t.slots, t.chunks, t.chunk, t.parts};
}
int check_table(const char* what, const niw_table* t, bool form_fits) {
    NIW_REQUIRE(t, "%s: null pointer", what);
    NIW_REQUIRE(form_fits, "%s: a table of form %d", what, t->form);
    NIW_REQUIRE(t->slots == 0 || (t->image && aligned(t->image, 16)), "%s: the table's image is not stored", what);
    return NIW_OK;
}

// The launch that leaves the partial sums of the list in `partial`; -> their number.  One partial sum is the total, and goes to `total` and
// `norm` (both may be null) at once.
template <class Slot>
int launch_partials(const List<Slot>& list, const niw_table& t, int kind, double* partial, double* total, float* norm, hipStream_t st) {
    const int grid = list.chunks < kNormBlocks ? list.chunks : kNormBlocks;
    if (grid == 0) return 0;
    const int cached = t.read <= kCache ? 0 : (int)((double)list.chunks * (1.0 - (double)kCache / (double)t.read));
    if (grid > 1) total = nullptr, norm = nullptr;
    if (kind == NIW_NORM_2) partial_kernel<NIW_NORM_2><<<grid, kThreads, 0, st>>>(list, cached, partial, total, norm);
    else partial_kernel<NIW_NORM_MAX><<<grid, kThreads, 0, st>>>(list, cached, partial, total, norm);
    return grid;
}
void launch_finish(int kind, const double* partial, int n, double* total, float* norm, hipStream_t st) {
    if (kind == NIW_NORM_2) finish_kernel<NIW_NORM_2><<<1, kThreads, 0, st>>>(partial, n, total, norm);
    else finish_kernel<NIW_NORM_MAX><<<1, kThreads, 0, st>>>(partial, n, total, norm);
}
template <class F>
void with_bool(bool value, F f) {
    if (value) f(std::true_type{});
    else f(std::false_type{});
}
// one workgroup per part (one for an empty list, whose norm is still written)
template <class Slot>
int64_t grid_of(const List<Slot>& list) {
    return list.chunks < 1 ? 1 : (int64_t)list.chunks * list.parts;
}
// the norm's launches in front of a kernel of `grid` workgroups that clips by it
template <class Slot>
void prepare_clip(Clip& clip, const List<Slot>& list, const niw_table& t, int64_t grid, int kind, const double* total, double* workspace, hipStream_t st) {
    clip.partial = total;
    clip.n_partial = 1;
    if (total) return;
    const int n = launch_partials(list, t, kind, workspace + 1, nullptr, nullptr, st);
    if (n > 0 && grid <= kFoldGrid) { clip.partial = workspace + 1; clip.n_partial = n; return; }
    launch_finish(kind, workspace + 1, n, workspace, nullptr, st);
    clip.partial = workspace;
}

}  // namespace

extern "C" int64_t niw_table_bytes(int64_t n_tensors) { return n_tensors < 0 ? 0 : padded((n_tensors + kMaxPieces) * (int64_t)(sizeof(AdamSlot) + sizeof(int))); }

extern "C" int niw_grad_table(const niw_grad_tensor* tensors, int64_t n_tensors, int flags, void* image, niw_table* table) try {
    NIW_REQUIRE(n_tensors >= 0 && n_tensors <= kMaxTensors && (tensors || n_tensors == 0), "niw_grad_table: %lld tensors at %p", (long long)n_tensors, (const void*)tensors);
    NIW_REQUIRE(table && (image || n_tensors == 0), "niw_grad_table: null pointer");
    NIW_REQUIRE((flags & ~(NIW_TABLE_CLIP | NIW_TABLE_KEPT)) == 0, "niw_grad_table: flags %d", flags);
    const bool for_clip = (flags & NIW_TABLE_CLIP) != 0;
    const int rc = check_grads("niw_grad_table", tensors, n_tensors, for_clip);
    return rc != NIW_OK ? rc : build<GradSlot>("niw_grad_table", tensors, n_tensors, for_clip ? kFormClip : kFormNorm, 0, (flags & NIW_TABLE_KEPT) != 0, image, table);
} catch (...) {
    niw_set_error("niw_grad_table: out of host memory");
    return NIW_ERR_INVALID_ARG;
}

extern "C" int niw_adam_table(const niw_adam_tensor* tensors, int64_t n_tensors, int n_groups, int flags, void* image, niw_table* table) try {
    NIW_REQUIRE(n_tensors >= 0 && n_tensors <= kMaxTensors && (tensors || n_tensors == 0), "niw_adam_table: %lld tensors at %p", (long long)n_tensors, (const void*)tensors);
    NIW_REQUIRE(table && (image || n_tensors == 0), "niw_adam_table: null pointer");
    NIW_REQUIRE((flags & ~NIW_TABLE_KEPT) == 0, "niw_adam_table: flags %d", flags);
    NIW_REQUIRE(n_groups >= 1 && n_groups <= NIW_ADAM_MAX_GROUPS, "niw_adam_table: 1..%d groups (got %d)", NIW_ADAM_MAX_GROUPS, n_groups);
    const int rc = check_adam("niw_adam_table", tensors, n_tensors, n_groups);
    return rc != NIW_OK ? rc : build<AdamSlot>("niw_adam_table", tensors, n_tensors, kFormAdam, n_groups, (flags & NIW_TABLE_KEPT) != 0, image, table);
} catch (...) {
    niw_set_error("niw_adam_table: out of host memory");
    return NIW_ERR_INVALID_ARG;
}

extern "C" int niw_table_store(const void* image, int64_t bytes, void* dst, niw_stream_t stream) {
    NIW_REQUIRE(bytes >= 0 && bytes % 16 == 0, "niw_table_store: %lld bytes", (long long)bytes);
    NIW_REQUIRE(bytes == 0 || (image && dst && aligned(dst, 16)), "niw_table_store: null or misaligned pointer");
    for (int64_t at = 0; at < bytes; at += sizeof(Piece)) {
        const int64_t size = bytes - at < (int64_t)sizeof(Piece) ? bytes - at : (int64_t)sizeof(Piece);
        Piece piece;
        memcpy(&piece, static_cast<const char*>(image) + at, size);
        store_kernel<<<1, kThreads, 0, (hipStream_t)stream>>>(piece, reinterpret_cast<u32x4*>(static_cast<char*>(dst) + at), (int)(size / 16));
    }
    NIW_LAUNCH_CHECK("niw_table_store");
    return NIW_OK;
}

extern "C" int niw_grad_norm(const niw_table* table, int kind, double* workspace, double* total, float* norm, niw_stream_t stream) {
    const int rc = check_table("niw_grad_norm", table, table && (table->form == kFormNorm || table->form == kFormClip));
    if (rc != NIW_OK) return rc;
    NIW_REQUIRE(kind == NIW_NORM_2 || kind == NIW_NORM_MAX, "niw_grad_norm: unknown kind %d", kind);
    NIW_REQUIRE(workspace && (total || norm), "niw_grad_norm: null pointer");
    hipStream_t st = (hipStream_t)stream;
    const int n = launch_partials(list_of<GradSlot>(*table), *table, kind, workspace + 1, total, norm, st);
    if (n != 1) launch_finish(kind, workspace + 1, n, total, norm, st);
    NIW_LAUNCH_CHECK("niw_grad_norm");
    return NIW_OK;
}

extern "C" int niw_grad_clip(const niw_table* table, int kind, double max_norm, const double* total, double* workspace, float* norm_out, niw_stream_t stream) {
    const int rc = check_table("niw_grad_clip", table, table && table->form == kFormClip);
    if (rc != NIW_OK) return rc;
    NIW_REQUIRE(kind == NIW_NORM_2 || kind == NIW_NORM_MAX, "niw_grad_clip: unknown kind %d", kind);
    NIW_REQUIRE(max_norm >= 0.0, "niw_grad_clip: max_norm=%g", max_norm);
    NIW_REQUIRE(workspace || total, "niw_grad_clip: null pointer");
    hipStream_t st = (hipStream_t)stream;
    const auto list = list_of<GradSlot>(*table);
    Clip clip{nullptr, norm_out, max_norm, 1, 0};
    const int64_t grid = grid_of(list);
    prepare_clip(clip, list, *table, grid, kind, total, workspace, st);
    with_bool(table->touched > kCache, [&](auto nt) {
        with_bool(table->wide != 0, [&](auto wide) {
            constexpr bool N = decltype(nt)::value;
            constexpr int P = decltype(wide)::value ? kClipPartWide : kClipPart;
            if (kind == NIW_NORM_2) clip_kernel<NIW_NORM_2, N, P><<<(unsigned)grid, kThreads, 0, st>>>(list, clip);
            else clip_kernel<NIW_NORM_MAX, N, P><<<(unsigned)grid, kThreads, 0, st>>>(list, clip);
        });
    });
    NIW_LAUNCH_CHECK("niw_grad_clip");
    return NIW_OK;
}

extern "C" int niw_adam_step_tensors(const niw_table* table, const niw_adam_hyper* hyper, double beta1, double beta2, double eps, const float* hyper_dev,
                                     const float* decay_dev, const niw_adam_clip* clip, niw_stream_t stream) {
    const int rc = check_table("niw_adam_step_tensors", table, table && table->form == kFormAdam);
    if (rc != NIW_OK) return rc;
    NIW_REQUIRE(hyper, "niw_adam_step_tensors: null pointer");
    NIW_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0, "niw_adam_step_tensors: beta1=%g beta2=%g eps=%g", beta1, beta2, eps);
    AdamArgs a{};
    bool decays = decay_dev != nullptr;
    for (int k = 0; k < table->groups; ++k) {
        const niw_adam_hyper& h = hyper[k];
        NIW_REQUIRE(h.step >= 1 || hyper_dev, "niw_adam_step_tensors: group %d step=%d", k, h.step);
        NIW_REQUIRE(isfinite(h.lr) && isfinite(h.weight_decay) && h.weight_decay >= 0.0, "niw_adam_step_tensors: group %d lr=%g weight_decay=%g", k, h.lr, h.weight_decay);
        NIW_REQUIRE(h.weight_decay == 0.0 || !hyper_dev || decay_dev, "niw_adam_step_tensors: group %d: weight_decay with hyper_dev needs decay_dev", k);
        const int step = h.step < 1 ? 1 : h.step;
        // the scalars are formed in double and rounded to fp32 once, as in niw_adam_step
        const double bc1 = 1.0 - pow(beta1, (double)step), bc2 = 1.0 - pow(beta2, (double)step);
        a.step_size[k] = (float)(h.lr / bc1);
        a.bc2_sqrt[k] = (float)sqrt(bc2);
        const float decay = (float)(h.lr * h.weight_decay);
        a.keep[k] = keep_of(decay);
        decays |= decay != 0.f;
    }
    a.w1 = (float)(1.0 - beta1); a.b2 = (float)beta2; a.w2 = (float)(1.0 - beta2); a.eps = (float)eps;
    a.hyper_dev = hyper_dev; a.decay_dev = decay_dev;
    hipStream_t st = (hipStream_t)stream;
    const auto list = list_of<AdamSlot>(*table);
    const int64_t grid = grid_of(list);
    Clip c{};
    if (clip) {
        NIW_REQUIRE(clip->kind == NIW_NORM_2 || clip->kind == NIW_NORM_MAX, "niw_adam_step_tensors: unknown kind %d", clip->kind);
        NIW_REQUIRE(clip->max_norm >= 0.0, "niw_adam_step_tensors: max_norm=%g", clip->max_norm);
        NIW_REQUIRE(clip->total || clip->workspace, "niw_adam_step_tensors: null pointer");
        c.norm_out = clip->norm; c.max_norm = clip->max_norm; c.skip_nonfinite = clip->skip_nonfinite;
        prepare_clip(c, list, *table, grid, clip->kind, clip->total, clip->workspace, st);
    }
    with_bool(table->touched > kCache, [&](auto nt) {
        with_bool(decays, [&](auto decay) {
            constexpr bool N = decltype(nt)::value, D = decltype(decay)::value;
            if (!clip || clip->kind == NIW_NORM_2) adam_tensors_kernel<NIW_NORM_2, N, D><<<(unsigned)grid, kThreads, 0, st>>>(list, a, c);
            else adam_tensors_kernel<NIW_NORM_MAX, N, D><<<(unsigned)grid, kThreads, 0, st>>>(list, a, c);
        });
    });
    NIW_LAUNCH_CHECK("niw_adam_step_tensors");
    return NIW_OK;
}
