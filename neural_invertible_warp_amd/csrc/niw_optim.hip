// The optimiser's end of a training step over a list of many tensors (include/niw.h):
//
//   niw_grad_norm           N = (sum_t sum_i g_ti^2)^(1/2), or max |g_ti|
//   niw_grad_clip           out = c g,  c = min(1, max_norm / (N + 1e-6))
//   niw_adam_step_tensors   Adam by c g, with decoupled weight decay, without ever writing c g
//
// All are streams of memory: 2 flops per element for the norm, 3 for clipping, about 18 for Adam.
//
// The list goes to the kernels BY VALUE, as many tensors per launch as 4 KB of kernel arguments hold (struct Table): no upload, no
// device table whose lifetime or stream somebody has to watch, and a captured graph carries its own copy.  A workgroup finds the
// tensor of its chunk by bisection over the chunks in front of each tensor (scalar loads of the argument segment).
//
// Sums.  A square of two 24-bit significands has 48 bits: it is exact in double, and so is its exponent for every fp32 value, so the
// sum of squares neither overflows (an fp32 sum does from |g| = 1.8e19) nor loses small gradients.  One fp64 fused multiply-add per
// element costs a quarter of what the memory stream leaves idle.  The maximum is taken over the bit patterns of |g| as integers,
// whose order is that of the values and puts NaN above infinity: a NaN is never dropped.
#include "niw_common.h"
#include "niw_bf16.h"
#include <math.h>
#include <algorithm>
#include <type_traits>
#include <vector>

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 16384;                 // elements of one tensor that one workgroup handles
constexpr double kClipEps = 1e-6;

// ------------------------------------------------------------------------------------------------ tables
struct GradSlot {
    const void* g;
    void* o;
    long long n;
    int first;                                // chunks of the tensors in front of this one in the launch
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
    int types;                                // param_dtype | grad_dtype << 8 | group << 16
};
template <class Slot, int N>
struct Table {
    Slot s[N];
    int count, chunks;
};
using GradTable = Table<GradSlot, 120>;
struct AdamTable : Table<AdamSlot, 64> {
    float step_size[NIW_ADAM_MAX_GROUPS], bc2_sqrt[NIW_ADAM_MAX_GROUPS], decay[NIW_ADAM_MAX_GROUPS];
    float w1, b2, w2, eps;
};
static_assert(sizeof(GradTable) <= 4000 && sizeof(AdamTable) <= 4000, "kernel arguments are limited to 4 KB");

// the tensor that chunk c of the launch belongs to
template <class T>
__device__ __forceinline__ int slot_of(const T& t, int c) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.s[mid].first <= c) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// ------------------------------------------------------------------------------------------------ elements
// Vectors of four elements (16 bytes of fp32, 8 of the half types) that may begin on any element: the aligned(..) attributes promise the
// compiler no more than that, and gfx950 takes such accesses as one instruction.
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));

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
template <int DT>
__device__ __forceinline__ f32x4 load4(const void* p, long long i) {
    if constexpr (DT == NIW_F32) return *reinterpret_cast<const f32x4_any*>(static_cast<const float*>(p) + i);
    else {
        const u32x2 w = *reinterpret_cast<const u32x2_any*>(static_cast<const unsigned short*>(p) + i);
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
template <int DT>
__device__ __forceinline__ void store4(void* p, long long i, f32x4 x) {
    if constexpr (DT == NIW_F32) *reinterpret_cast<f32x4_any*>(static_cast<float*>(p) + i) = x;
    else *reinterpret_cast<u32x2_any*>(static_cast<unsigned short*>(p) + i) = u32x2{narrow2<DT>(x[0], x[1]), narrow2<DT>(x[2], x[3])};
}
// f(std::integral_constant dtype) for the dtype of a descriptor: the branch is the same for a whole workgroup
template <class F>
__device__ __forceinline__ void with_dtype(int dtype, F f) {
    if (dtype == NIW_F32) f(std::integral_constant<int, NIW_F32>{});
    else if (dtype == NIW_BF16) f(std::integral_constant<int, NIW_BF16>{});
    else f(std::integral_constant<int, NIW_F16>{});
}

// ------------------------------------------------------------------------------------------------ reductions
// accumulators: the sum of squares as a double, the maximum as the integer bits of |g| held in a double's place
template <int KIND>
__device__ __forceinline__ double join(double a, double b) {
    if constexpr (KIND == NIW_NORM_2) return a + b;
    else return a != a ? a : (b != b ? b : (a > b ? a : b));
}
template <int KIND>
__device__ __forceinline__ double block_total(double x) {
    __shared__ double part[16];
#pragma unroll
    for (int m = 32; m; m >>= 1) x = join<KIND>(x, __shfl_xor(x, m, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = part[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) x = join<KIND>(x, part[w]);
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
template <int KIND, int DT>
__device__ __forceinline__ void see(Seen<KIND>& seen, const void* p, long long begin, long long end) {
    constexpr int V = DT == NIW_F32 ? 4 : 8, U = 4;      // 16 bytes per thread and load, U loads under way
    const int tid = threadIdx.x;
    auto words = [&](long long i) { return *reinterpret_cast<const u32x4_any*>(static_cast<const char*>(p) + i * (16 / V)); };
    auto take = [&](u32x4 w) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned bits = w[k];          // (a copy: clang's bit_cast of a vector element in place reads element 0)
            if constexpr (DT == NIW_F32) seen(k, __builtin_bit_cast(float, bits));
            else { seen(2 * k, widen<DT>((unsigned short)bits)); seen(2 * k + 1, widen<DT>((unsigned short)(bits >> 16))); }
        }
    };
    long long i = begin;
    for (; i + (long long)kThreads * V * U <= end; i += (long long)kThreads * V * U) {
        u32x4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = words(i + (u * kThreads + tid) * V);
#pragma unroll
        for (int u = 0; u < U; ++u) take(w[u]);
    }
    for (i += tid * V; i + V <= end; i += kThreads * V) take(words(i));
    if (i < end)
        for (; i < end; ++i) seen(0, load1<DT>(p, i));
}

template <int KIND>
__global__ __launch_bounds__(kThreads) void partial_kernel(GradTable t, double* __restrict__ partial) {
    const GradSlot& s = t.s[slot_of(t, blockIdx.x)];
    const long long begin = (long long)((int)blockIdx.x - s.first) * kChunk, end = begin + kChunk < s.n ? begin + kChunk : s.n;
    Seen<KIND> seen;
    with_dtype(s.types & 255, [&](auto dt) { see<KIND, decltype(dt)::value>(seen, s.g, begin, end); });
    const double sum = block_total<KIND>(seen.total());
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

__device__ __forceinline__ double norm_of(double total, int kind) { return kind == NIW_NORM_2 ? sqrt(total) : total; }

template <int KIND>
__global__ __launch_bounds__(1024) void finish_kernel(const double* __restrict__ partial, long long n, double* __restrict__ total, float* __restrict__ norm) {
    double x = 0.0;
    for (long long i = threadIdx.x; i < n; i += 1024) x = join<KIND>(x, partial[i]);
    x = block_total<KIND>(x);
    if (threadIdx.x == 0) {
        if (total) total[0] = x;
        if (norm) norm[0] = (float)norm_of(x, KIND);
    }
}

__device__ __forceinline__ float clip_factor(double norm, double max_norm) {
    if (isinf(max_norm)) return 1.f;
    const double c = max_norm / (norm + kClipEps);
    return c < 1.0 ? (float)c : (c != c ? (float)c : 1.f);
}

__global__ __launch_bounds__(kThreads) void clip_kernel(GradTable t, const double* __restrict__ total, int kind, double max_norm, float* __restrict__ norm_out) {
    const double norm = norm_of(total[0], kind);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = (float)norm;
    if (t.count == 0) return;
    const float c = clip_factor(norm, max_norm);
    const GradSlot& s = t.s[slot_of(t, blockIdx.x)];
    if (c == 1.f && s.o == s.g) return;
    const long long begin = (long long)((int)blockIdx.x - s.first) * kChunk, end = begin + kChunk < s.n ? begin + kChunk : s.n;
    with_dtype(s.types & 255, [&](auto gt) {
        with_dtype(s.types >> 8, [&](auto ot) {
            constexpr int G = decltype(gt)::value, O = decltype(ot)::value, U = 4;
            long long i = begin;
            for (; i + kThreads * 4 * U <= end; i += kThreads * 4 * U) {
                f32x4 x[U];
#pragma unroll
                for (int u = 0; u < U; ++u) x[u] = load4<G>(s.g, i + (u * kThreads + (int)threadIdx.x) * 4);
#pragma unroll
                for (int u = 0; u < U; ++u) store4<O>(s.o, i + (u * kThreads + (int)threadIdx.x) * 4, c * x[u]);
            }
            for (i += (int)threadIdx.x * 4; i + 4 <= end; i += kThreads * 4) store4<O>(s.o, i, c * load4<G>(s.g, i));
            if (i < end)
                for (; i < end; ++i) store1<O>(s.o, i, c * load1<G>(s.g, i));
        });
    });
}

__global__ __launch_bounds__(kThreads) void adam_tensors_kernel(AdamTable t, const float* __restrict__ hyper_dev, const float* __restrict__ decay_dev,
                                                                const double* __restrict__ total, int kind, int skip_nonfinite, double max_norm,
                                                                float* __restrict__ norm_out) {
    float c = 1.f;
    if (total) {
        const double norm = norm_of(total[0], kind);
        if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = (float)norm;
        if (skip_nonfinite && !isfinite(norm)) return;
        c = clip_factor(norm, max_norm);
    }
    if (t.count == 0) return;
    const AdamSlot& s = t.s[slot_of(t, blockIdx.x)];
    const int param_dtype = s.types & 255, grad_dtype = (s.types >> 8) & 255, k = s.types >> 16;
    float step_size = t.step_size[k], bc2_sqrt = t.bc2_sqrt[k], decay = t.decay[k];
    if (hyper_dev) { step_size = hyper_dev[2 * k]; bc2_sqrt = hyper_dev[2 * k + 1]; }
    if (decay_dev) decay = decay_dev[k];
    const long long begin = (long long)((int)blockIdx.x - s.first) * kChunk, end = begin + kChunk < s.n ? begin + kChunk : s.n;
    float* const w = s.w ? s.w : static_cast<float*>(s.p);
    auto update = [&](float& p, float g, float& m, float& v) {
        p = fmaf(-decay, p, p);
        niw::adam_update(p, niw::mul_rn(c, g), m, v, t.w1, t.b2, t.w2, t.eps, step_size, bc2_sqrt);
    };
    with_dtype(grad_dtype, [&](auto gt) {
        with_dtype(param_dtype, [&](auto pt) {
            constexpr int G = decltype(gt)::value, P = decltype(pt)::value;
            long long i = begin + (int)threadIdx.x * 4;
            for (; i + 4 <= end; i += kThreads * 4) {
                f32x4 p = load4<NIW_F32>(w, i), m = load4<NIW_F32>(s.m, i), v = load4<NIW_F32>(s.v, i);
                const f32x4 g = load4<G>(s.g, i);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float pk = p[k], mk = m[k], vk = v[k];
                    update(pk, g[k], mk, vk);
                    p[k] = pk; m[k] = mk; v[k] = vk;
                }
                store4<NIW_F32>(w, i, p);
                store4<NIW_F32>(s.m, i, m);
                store4<NIW_F32>(s.v, i, v);
                if constexpr (P != NIW_F32) store4<P>(s.p, i, p);
            }
            for (; i < end; ++i) {
                float p = w[i], m = s.m[i], v = s.v[i];
                update(p, load1<G>(s.g, i), m, v);
                w[i] = p; s.m[i] = m; s.v[i] = v;
                if constexpr (P != NIW_F32) store1<P>(s.p, i, p);
            }
        });
    });
}

// ------------------------------------------------------------------------------------------------ host
int size_of(int dtype) { return dtype == NIW_F32 ? 4 : 2; }
bool known(int dtype) { return dtype == NIW_F32 || dtype == NIW_BF16 || dtype == NIW_F16; }
bool aligned(const void* p, int size) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(size - 1)) == 0; }
long long chunks_of(long long n) { return (n + kChunk - 1) / kChunk; }
constexpr int64_t kMaxElements = 1ll << 44;   // (chunks of one tensor stay far below 2^31)

int check_grads(const char* what, const niw_grad_tensor* t, int64_t count, bool for_clip) {
    NIW_REQUIRE(count >= 0 && (t || count == 0), "%s: %lld tensors at a null pointer", what, (long long)count);
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
    return NIW_OK;
}

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

// calls f(table, chunks of the launches before it) for the launches that `count` tensors take; tensors without elements are left out
template <class T, class Item, class Fill, class Launch>
int for_tables(const Item* items, int64_t count, T& table, Fill fill, Launch launch) {
    constexpr int kSlots = sizeof(table.s) / sizeof(table.s[0]);
    long long before = 0;
    table.count = table.chunks = 0;
    for (int64_t i = 0; i < count; ++i) {
        if (items[i].n == 0) continue;
        const long long chunks = chunks_of(items[i].n);
        if (table.count == kSlots || table.chunks + chunks > 0x7fffffffll) {
            const int rc = launch(table, before);
            if (rc != NIW_OK) return rc;
            before += table.chunks;
            table.count = table.chunks = 0;
        }
        fill(table.s[table.count], items[i]);
        table.s[table.count].first = table.chunks;
        ++table.count;
        table.chunks += (int)chunks;
    }
    return table.count ? launch(table, before) : NIW_OK;
}

// the list's total into `total` (and the norm): partial sums of every launch, then one workgroup over them
template <class Item, class Fill>
int total_of(const char* what, const Item* items, int64_t count, Fill fill, int kind, double* workspace, double* total, float* norm, hipStream_t st) {
    GradTable table{};
    long long partials = 0;
    const int rc = for_tables(items, count, table, fill, [&](const GradTable& t, long long before) -> int {
        if (kind == NIW_NORM_2) partial_kernel<NIW_NORM_2><<<t.chunks, kThreads, 0, st>>>(t, workspace + before);
        else partial_kernel<NIW_NORM_MAX><<<t.chunks, kThreads, 0, st>>>(t, workspace + before);
        partials = before + t.chunks;
        NIW_LAUNCH_CHECK(what);
        return NIW_OK;
    });
    if (rc != NIW_OK) return rc;
    if (kind == NIW_NORM_2) finish_kernel<NIW_NORM_2><<<1, 1024, 0, st>>>(workspace, partials, total, norm);
    else finish_kernel<NIW_NORM_MAX><<<1, 1024, 0, st>>>(workspace, partials, total, norm);
    NIW_LAUNCH_CHECK(what);
    return NIW_OK;
}

template <class Item>
int64_t workspace_doubles(const Item* t, int64_t count) {
    long long n = 1;                          // the total stands in front of the partial sums
    for (int64_t i = 0; t && i < count; ++i) n += t[i].n > 0 ? chunks_of(t[i].n) : 0;
    return n;
}

void fill_grad(GradSlot& s, const niw_grad_tensor& t) {
    s.g = t.grad; s.o = t.out; s.n = t.n; s.types = t.dtype | t.out_dtype << 8;
}
void fill_adam_grad(GradSlot& s, const niw_adam_tensor& t) {
    s.g = t.grad; s.o = nullptr; s.n = t.n; s.types = t.grad_dtype;
}
void fill_adam(AdamSlot& s, const niw_adam_tensor& t) {
    s.p = t.param; s.g = t.grad; s.m = t.exp_avg; s.v = t.exp_avg_sq; s.w = t.master; s.n = t.n;
    s.types = t.param_dtype | t.grad_dtype << 8 | t.group << 16;
}

int check_adam(const char* what, const niw_adam_tensor* t, int64_t count, int n_groups) {
    NIW_REQUIRE(count >= 0 && (t || count == 0), "%s: %lld tensors at a null pointer", what, (long long)count);
    NIW_REQUIRE(n_groups >= 1 && n_groups <= NIW_ADAM_MAX_GROUPS, "%s: 1..%d groups (got %d)", what, NIW_ADAM_MAX_GROUPS, n_groups);
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
    return NIW_OK;
}

}  // namespace

extern "C" int niw_grad_check(const niw_grad_tensor* tensors, int64_t n_tensors, int for_clip) {
    const int rc = check_grads("niw_grad_check", tensors, n_tensors, for_clip != 0);
    if (rc != NIW_OK || !for_clip) return rc;
    try {
        std::vector<Range> r;
        r.reserve(2 * n_tensors);
        for (int64_t i = 0; i < n_tensors; ++i) {
            const niw_grad_tensor& t = tensors[i];
            if (t.out != t.grad) add_range(r, t.grad, t.n, size_of(t.dtype), i, false);
            add_range(r, t.out, t.n, size_of(t.out_dtype), i, true);
        }
        return check_overlaps("niw_grad_check", r);
    } catch (...) {
        niw_set_error("niw_grad_check: out of host memory");
        return NIW_ERR_INVALID_ARG;
    }
}

extern "C" int64_t niw_grad_workspace_doubles(const niw_grad_tensor* tensors, int64_t n_tensors) { return workspace_doubles(tensors, n_tensors); }

extern "C" int niw_grad_norm(const niw_grad_tensor* tensors, int64_t n_tensors, int kind, double* workspace, double* total, float* norm, niw_stream_t stream) {
    const int rc = check_grads("niw_grad_norm", tensors, n_tensors, false);
    if (rc != NIW_OK) return rc;
    NIW_REQUIRE(kind == NIW_NORM_2 || kind == NIW_NORM_MAX, "niw_grad_norm: unknown kind %d", kind);
    NIW_REQUIRE(workspace && (total || norm), "niw_grad_norm: null pointer");
    return total_of("niw_grad_norm", tensors, n_tensors, fill_grad, kind, workspace + 1, total, norm, (hipStream_t)stream);
}

extern "C" int niw_grad_clip(const niw_grad_tensor* tensors, int64_t n_tensors, int kind, double max_norm, const double* total, double* workspace,
                             float* norm_out, niw_stream_t stream) {
    int rc = check_grads("niw_grad_clip", tensors, n_tensors, true);
    if (rc != NIW_OK) return rc;
    NIW_REQUIRE(kind == NIW_NORM_2 || kind == NIW_NORM_MAX, "niw_grad_clip: unknown kind %d", kind);
    NIW_REQUIRE(max_norm >= 0.0, "niw_grad_clip: max_norm=%g", max_norm);
    NIW_REQUIRE(workspace || total, "niw_grad_clip: null pointer");
    hipStream_t st = (hipStream_t)stream;
    if (!total) {
        rc = total_of("niw_grad_clip", tensors, n_tensors, fill_grad, kind, workspace + 1, workspace, nullptr, st);
        if (rc != NIW_OK) return rc;
        total = workspace;
    }
    GradTable table{};
    bool launched = false;
    rc = for_tables(tensors, n_tensors, table, fill_grad, [&](const GradTable& t, long long) -> int {
        clip_kernel<<<t.chunks, kThreads, 0, st>>>(t, total, kind, max_norm, launched ? nullptr : norm_out);
        launched = true;
        NIW_LAUNCH_CHECK("niw_grad_clip");
        return NIW_OK;
    });
    if (rc != NIW_OK || launched || !norm_out) return rc;
    clip_kernel<<<1, kThreads, 0, st>>>(table, total, kind, max_norm, norm_out);      // (an empty list: the norm alone)
    NIW_LAUNCH_CHECK("niw_grad_clip");
    return NIW_OK;
}

extern "C" int niw_adam_check(const niw_adam_tensor* tensors, int64_t n_tensors, int n_groups) {
    const int rc = check_adam("niw_adam_check", tensors, n_tensors, n_groups);
    if (rc != NIW_OK) return rc;
    try {
        std::vector<Range> r;
        r.reserve(5 * n_tensors);
        for (int64_t i = 0; i < n_tensors; ++i) {
            const niw_adam_tensor& t = tensors[i];
            add_range(r, t.param, t.n, size_of(t.param_dtype), i, true);
            add_range(r, t.grad, t.n, size_of(t.grad_dtype), i, false);
            add_range(r, t.exp_avg, t.n, 4, i, true);
            add_range(r, t.exp_avg_sq, t.n, 4, i, true);
            if (t.master) add_range(r, t.master, t.n, 4, i, true);
        }
        return check_overlaps("niw_adam_check", r);
    } catch (...) {
        niw_set_error("niw_adam_check: out of host memory");
        return NIW_ERR_INVALID_ARG;
    }
}

extern "C" int64_t niw_adam_workspace_doubles(const niw_adam_tensor* tensors, int64_t n_tensors) { return workspace_doubles(tensors, n_tensors); }

extern "C" int niw_adam_step_tensors(const niw_adam_tensor* tensors, int64_t n_tensors, const niw_adam_hyper* hyper, int n_groups, double beta1, double beta2,
                                     double eps, const float* hyper_dev, const float* decay_dev, const niw_adam_clip* clip, niw_stream_t stream) {
    int rc = check_adam("niw_adam_step_tensors", tensors, n_tensors, n_groups);
    if (rc != NIW_OK) return rc;
    NIW_REQUIRE(hyper, "niw_adam_step_tensors: null pointer");
    NIW_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0, "niw_adam_step_tensors: beta1=%g beta2=%g eps=%g", beta1, beta2, eps);
    AdamTable table{};
    for (int k = 0; k < n_groups; ++k) {
        const niw_adam_hyper& h = hyper[k];
        NIW_REQUIRE(h.step >= 1 || hyper_dev, "niw_adam_step_tensors: group %d step=%d", k, h.step);
        NIW_REQUIRE(isfinite(h.lr) && isfinite(h.weight_decay) && h.weight_decay >= 0.0, "niw_adam_step_tensors: group %d lr=%g weight_decay=%g", k, h.lr, h.weight_decay);
        NIW_REQUIRE(h.weight_decay == 0.0 || !hyper_dev || decay_dev, "niw_adam_step_tensors: group %d: weight_decay with hyper_dev needs decay_dev", k);
        const int step = h.step < 1 ? 1 : h.step;
        // the scalars are formed in double and rounded to fp32 once, as in niw_adam_step
        const double bc1 = 1.0 - pow(beta1, (double)step), bc2 = 1.0 - pow(beta2, (double)step);
        table.step_size[k] = (float)(h.lr / bc1);
        table.bc2_sqrt[k] = (float)sqrt(bc2);
        table.decay[k] = (float)(h.lr * h.weight_decay);
    }
    table.w1 = (float)(1.0 - beta1); table.b2 = (float)beta2; table.w2 = (float)(1.0 - beta2); table.eps = (float)eps;
    hipStream_t st = (hipStream_t)stream;
    const double* total = nullptr;
    if (clip) {
        NIW_REQUIRE(clip->kind == NIW_NORM_2 || clip->kind == NIW_NORM_MAX, "niw_adam_step_tensors: unknown kind %d", clip->kind);
        NIW_REQUIRE(clip->max_norm >= 0.0, "niw_adam_step_tensors: max_norm=%g", clip->max_norm);
        NIW_REQUIRE(clip->total || clip->workspace, "niw_adam_step_tensors: null pointer");
        total = clip->total;
        if (!total) {
            rc = total_of("niw_adam_step_tensors", tensors, n_tensors, fill_adam_grad, clip->kind, clip->workspace + 1, clip->workspace, nullptr, st);
            if (rc != NIW_OK) return rc;
            total = clip->workspace;
        }
    }
    const int kind = clip ? clip->kind : 0, skip = clip ? clip->skip_nonfinite : 0;
    const double max_norm = clip ? clip->max_norm : 0.0;
    float* const norm_out = clip ? clip->norm : nullptr;
    bool launched = false;
    rc = for_tables(tensors, n_tensors, table, fill_adam, [&](const AdamTable& t, long long) -> int {
        adam_tensors_kernel<<<t.chunks, kThreads, 0, st>>>(t, hyper_dev, decay_dev, total, kind, skip, max_norm, launched ? nullptr : norm_out);
        launched = true;
        NIW_LAUNCH_CHECK("niw_adam_step_tensors");
        return NIW_OK;
    });
    if (rc != NIW_OK || launched || !norm_out) return rc;
    adam_tensors_kernel<<<1, kThreads, 0, st>>>(table, hyper_dev, decay_dev, total, kind, skip, max_norm, norm_out);      // (an empty list: the norm alone)
    NIW_LAUNCH_CHECK("niw_adam_step_tensors");
    return NIW_OK;
}
