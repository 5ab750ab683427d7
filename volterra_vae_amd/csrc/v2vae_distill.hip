// Distillation from a teacher's top logits: loss, gradient, or both in one pass over the student's logits.
//
// Row by row: with s = z / T,  m = max s,  l = sum exp(s - m),  q = exp(s - m) / l;  over the k teacher entries p = softmax(t / T),
// loss = T^2 sum_j p_j (log p_j - (s_j - m - log l)),  dz = w T (q - p at its classes).  The dense part is bound by reading z and
// writing dz once: a row is held in registers between the maximum, the sum and the gradient where it fits, by a group of lanes of
// one wave (short rows) or by a whole workgroup (long ones); longer rows still are read again, out of the caches.  The k
// sparse terms are patched over the dense gradient afterwards by the threads that hold the entries; a class that a row names
// twice is patched by the first of its entries with the sum, so no two threads write one address and no atomics are needed.
//
// Float 262144 x 64, 8 entries: loss 26 us (3.2 TB/s), gradient 35 (4.4 TB/s), both in one pass 38 ... 41: short rows are bound by issue, the
// vector instructions take a SIMD 24, 29 and 36 us of them.  bf16 4096 x 32000, 64 entries, loss and gradient 125 us (4.2 TB/s; a large
// copy: 5.2); f16 33 x 65521 loss 7.8 us, the time of one row's loads and reductions.  Measured and not kept: 256
// threads of sixteen pieces instead of 512 of eight (no change).
#include <math.h>

#include "v2vae_dense.h"

namespace v2vae {

struct DistillArgs {
    const void* z;
    const void* t;
    const void* index;
    const float* weight;  // [rows], gradient weight
    float* loss;          // [rows] or NULL
    float* stats;         // [rows][2]: written by the loss pass, read by the gradient pass
    void* grad;           // [rows][V] or NULL
    int64_t ld_z, ld_t, ld_i;
    int64_t rows;
    int V, k, teacher_dtype, wide_index;
    float inv_t, T;
};

enum { DO_LOSS = 1, DO_GRAD = 2 };

__device__ __forceinline__ float teacher_at(const DistillArgs& a, int64_t row, int j) {
    const int64_t o = row * a.ld_t + j;
    return a.teacher_dtype == V2VAE_F32 ? ((const float*)a.t)[o]
           : a.teacher_dtype == V2VAE_BF16 ? (float)((const bf16_t*)a.t)[o] : (float)((const f16_t*)a.t)[o];
}
// class of entry j: -1 absent, -2 beyond the vocabulary
__device__ __forceinline__ int class_at(const DistillArgs& a, int64_t row, int j) {
    const int64_t o = row * a.ld_i + j;
    const int64_t c = a.wide_index ? ((const int64_t*)a.index)[o] : (int64_t)((const int32_t*)a.index)[o];
    return c < 0 ? -1 : c >= a.V ? -2 : (int)c;
}

// Reductions over the lanes of a group: G lanes of a wave, or all threads of a workgroup through LDS (one barrier: every reduction of
// a kernel has a slot of its own).  Every lane gets the result; the order is fixed.
template <int G> struct Lanes {
    float* scratch;
    template <typename F> __device__ __forceinline__ float join(float v, int slot, F f) const {
#pragma unroll
        for (int d = (G < 64 ? G : 64) / 2; d > 0; d >>= 1) v = f(v, __shfl_xor(v, d));
        if constexpr (G > 64) {
            float* const at = scratch + slot * (G / 64);
            if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
            __syncthreads();
            v = at[0];
#pragma unroll
            for (int i = 1; i < G / 64; ++i) v = f(v, at[i]);
        }
        return v;
    }
    __device__ __forceinline__ float max(float v, int slot) const {
        return join(v, slot, [](float x, float y) { return fmaxf(x, y); });
    }
    __device__ __forceinline__ float sum(float v, int slot) const {
        return join(v, slot, [](float x, float y) { return x + y; });
    }
    __device__ __forceinline__ void sync() const {
        if constexpr (G > 64) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    }
};

constexpr float LOG2E = 1.4426950408889634f;
// exp((z - m) / T) for c = log2(e) / T: the difference first (exact where it matters, finite for the type's lowest values), then the
// base-2 exponential of the hardware
__device__ __forceinline__ float exp_diff(float z, float m, float c) { return __builtin_amdgcn_exp2f((z - m) * c); }

// G lanes a row, NV 16-byte pieces of the row held by each lane (HELD), or the row read once per pass.  MODE: DO_LOSS | DO_GRAD.
// A DO_GRAD pass alone takes maximum and sum from `stats`.  ONE: the teacher's entries fit the lanes of one wave (k <= G and
// k <= 64): each of them keeps one, and everything about them happens there while the row is on its way.  Else they are dealt out
// to the threads of the workgroup, their classes and probabilities in LDS for the merging of what names one class twice.
template <typename T, int G, int NV, bool HELD, int MODE, bool ONE>
__global__ __launch_bounds__(G > 64 ? G : 256) void k_distill(DistillArgs a) {
    constexpr int E = Vec16<T>::N, ROWS = G > 64 ? 1 : 256 / G, GE = G > 64 ? 64 : G;
    constexpr bool STATS_GIVEN = MODE == DO_GRAD;
    static_assert(ONE || G > 64, "lists need a workgroup");
    __shared__ float s_red[G > 64 ? 5 * (G / 64) : 1];
    __shared__ int s_state;
    __shared__ float s_p[ONE ? 1 : V2VAE_DISTILL_MAX_K];
    __shared__ int s_c[ONE ? 1 : V2VAE_DISTILL_MAX_K];
    const Lanes<G> lanes{s_red};
    const Lanes<GE> wave{nullptr};
    const int tid = G > 64 ? threadIdx.x : threadIdx.x % G;
    const int64_t row = (int64_t)blockIdx.x * ROWS + (G > 64 ? 0 : threadIdx.x / G);
    if (row >= a.rows) return;  // G > 64: a workgroup has one row; G <= 64: whole groups leave, shuffles stay within a group
    const T* const z = (const T*)a.z + row * a.ld_z;
    // pieces are cut at 16-byte addresses: `off` elements of the first piece lie before the row
    const int off = (int)(((uintptr_t)z & 15) / sizeof(T));
    const T* const z0 = z - off;
    const int pieces = (a.V + off + E - 1) / E;
    auto get = [&](int i) {
        Vec16<T> v;
        const int lo = i * E - off;
        if (lo >= 0 && lo + E <= a.V) {
            v.raw = *reinterpret_cast<const u32x4*>(z0 + i * E);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v.e[e] = (lo + e >= 0 && lo + e < a.V) ? z[lo + e] : (T)(-INFINITY);
        }
        return v;
    };
    const float c = a.inv_t * LOG2E;
    auto finite = [](float m) { return m == -INFINITY ? 0.f : m; };

    Vec16<T> raw[HELD ? NV : 1];
    if constexpr (HELD) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (tid + i * G < pieces) raw[i] = get(tid + i * G);
    }

    // The teacher's entries: p = softmax over the present ones.  ONE: lane j has entry j; p_all and `first` merge what names one
    // class twice.
    enum { NOTHING, SOME, BAD };
    int state = NOTHING, my_cls = -1;
    float my_p = 0.f, my_lp = 0.f, my_z = 0.f, p_all = 0.f, tmax = -INFINITY, inv_mass = 0.f, log_mass = 0.f;
    bool first = true;
    if constexpr (ONE) {
        if (tid < GE) {
            float t = -INFINITY;
            if (tid < a.k) {
                my_cls = class_at(a, row, tid);
                t = teacher_at(a, row, tid);
                if (my_cls >= 0) my_z = (float)z[my_cls];
            }
            // a class beyond the vocabulary, a NaN: as +inf, which makes the row NaN
            tmax = wave.max(my_cls == -2 || (my_cls >= 0 && t != t) ? INFINITY : my_cls >= 0 ? t : -INFINITY, 0);
            state = tmax == INFINITY ? BAD : tmax == -INFINITY ? NOTHING : SOME;
            const float lt = (t - tmax) * a.inv_t, e = my_cls >= 0 && state == SOME ? expf(lt) : 0.f;
            const float mass = wave.sum(e, 0);
            if (state == SOME) {
                my_p = e / mass;
                my_lp = lt - logf(mass);
            }
            if constexpr (MODE & DO_GRAD) {
                for (int i = 0; i < a.k; ++i) {  // all lanes of the group, entry or not
                    int ci;
                    float pi;
                    if constexpr (GE == 64) {  // a whole wave: lane i's registers are read as scalars, without LDS
                        ci = __builtin_amdgcn_readlane(my_cls, i);
                        pi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_p), i));
                    } else {
                        ci = __shfl(my_cls, i, GE);
                        pi = __shfl(my_p, i, GE);
                    }
                    if (ci == my_cls) {
                        p_all += pi;
                        first &= i >= tid;
                    }
                }
            }
            if (G > 64 && tid == 0) s_state = state;  // read behind the barriers below
        }
    }

    // the row: logits, then their exponentials in place
    float held[HELD ? NV : 1][E];
    float zmax = -INFINITY, l = 0.f;
    if constexpr (HELD) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) held[i][e] = tid + i * G < pieces ? (float)raw[i].e[e] : -INFINITY;
    }
    if constexpr (!STATS_GIVEN) {
        if constexpr (HELD) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) zmax = fmaxf(zmax, held[i][e]);
            zmax = lanes.max(zmax, 0);
            const float zm = finite(zmax);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    held[i][e] = exp_diff(held[i][e], zm, c);
                    l += held[i][e];
                }
            l = lanes.sum(l, 1);
        } else {
            // one pass with a running maximum per thread, joined at the end; NV pieces in flight
            float mine = -INFINITY;
            for (int i0 = tid; i0 < pieces; i0 += NV * G) {
                Vec16<T> v[NV];
#pragma unroll
                for (int i = 0; i < NV; ++i) v[i] = get(i0 + i * G);
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < E; ++e) top = fmaxf(top, (float)v[i].e[e]);
                if (top > mine) {
                    l *= exp_diff(mine, top, c);
                    mine = top;
                }
                const float at = finite(mine);
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < E; ++e) l += exp_diff((float)v[i].e[e], at, c);
            }
            zmax = lanes.max(mine, 0);
            l = lanes.sum(mine == -INFINITY ? l : l * exp_diff(mine, zmax, c), 1);
        }
        if (a.stats && tid == 0) {
            a.stats[2 * row] = zmax;
            a.stats[2 * row + 1] = l;
        }
    } else {
        zmax = a.stats[2 * row];
        l = a.stats[2 * row + 1];
        if constexpr (G > 64 && ONE) __syncthreads();
    }
    const float zm = finite(zmax), log_l = logf(l);
    if constexpr (G > 64 && ONE) state = s_state;

    if constexpr (!ONE) {
        int bad = 0;
        for (int j = tid; j < a.k; j += G) {
            const int cls = class_at(a, row, j);
            const float t = teacher_at(a, row, j);
            bad |= cls == -2 || (cls >= 0 && t != t);
            if (cls >= 0) tmax = fmaxf(tmax, t);
        }
        tmax = lanes.max(bad ? INFINITY : tmax, 2);
        state = tmax == INFINITY ? BAD : tmax == -INFINITY ? NOTHING : SOME;
        float mass = 0.f;
        for (int j = tid; j < a.k && state == SOME; j += G)
            if (class_at(a, row, j) >= 0) mass += expf((teacher_at(a, row, j) - tmax) * a.inv_t);
        mass = lanes.sum(mass, 3);
        if (state == SOME) {
            inv_mass = 1.f / mass;
            log_mass = logf(mass);
        }
    }
    auto entry_p = [&](int j, int cls) { return cls >= 0 && state == SOME ? expf((teacher_at(a, row, j) - tmax) * a.inv_t) * inv_mass : 0.f; };
    auto entry_loss = [&](float p, float lp, float zj) {  // p (log p - log q)
        return p == 0.f ? 0.f : p * (lp - (zj == -INFINITY ? -INFINITY : (zj - zm) * a.inv_t - log_l));
    };

    if constexpr (MODE & DO_LOSS) {
        float loss = 0.f;
        if constexpr (ONE) {
            if (tid < GE) loss = wave.sum(entry_loss(my_p, my_lp, my_z), 0);
        } else {
            for (int j = tid; j < a.k && state == SOME; j += G) {
                const int cls = class_at(a, row, j);
                const float p = entry_p(j, cls);
                if (p != 0.f) loss += entry_loss(p, (teacher_at(a, row, j) - tmax) * a.inv_t - log_mass, (float)z[cls]);
            }
            loss = lanes.sum(loss, 4);
        }
        if (tid == 0) a.loss[row] = state == BAD ? NAN : a.T * a.T * loss;
    }
    if constexpr (MODE & DO_GRAD) {
        const float wt = state == BAD ? NAN : a.weight[row] * a.T;
        const bool live = state != NOTHING;
        const float inv_l = l == 0.f ? 0.f : 1.f / l, scale = wt * inv_l;
        T* const out = (T*)a.grad + row * a.V;
        const bool same_phase = (int)(((uintptr_t)out & 15) / sizeof(T)) == off;
        auto put = [&](int i, const float (&v)[E]) {  // exponentials of piece i
            Vec16<T> o;
#pragma unroll
            for (int e = 0; e < E; ++e) o.e[e] = (T)(live ? v[e] * scale : 0.f);
            const int lo = i * E - off;
            if (same_phase && lo >= 0 && lo + E <= a.V) {
                *reinterpret_cast<u32x4*>(out + lo) = o.raw;
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (lo + e >= 0 && lo + e < a.V) out[lo + e] = o.e[e];
            }
        };
        if constexpr (HELD) {
            if constexpr (STATS_GIVEN) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < E; ++e) held[i][e] = exp_diff(held[i][e], zm, c);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (tid + i * G < pieces) put(tid + i * G, held[i]);
        } else {
            for (int i = tid; i < pieces; i += G) {
                const Vec16<T> v = get(i);
                float ev[E];
#pragma unroll
                for (int e = 0; e < E; ++e) ev[e] = exp_diff((float)v.e[e], zm, c);
                put(i, ev);
            }
        }
        if constexpr (!ONE) {
            for (int j = tid; j < a.k; j += G) {
                s_c[j] = class_at(a, row, j);
                s_p[j] = entry_p(j, s_c[j]);
            }
        }
        lanes.sync();
        if constexpr (ONE) {
            if (my_cls >= 0 && state == SOME && first) out[my_cls] = (T)(wt * (exp_diff(my_z, zm, c) * inv_l - p_all));
        } else {
            for (int j = tid; j < a.k; j += G) {
                const int cls = s_c[j];
                if (cls < 0 || state != SOME) continue;
                float p = 0.f;
                bool one = true;
                for (int i = 0; i < a.k; ++i) {
                    if (s_c[i] == cls) {
                        p += s_p[i];
                        one &= i >= j;
                    }
                }
                if (one) out[cls] = (T)(wt * (exp_diff((float)z[cls], zm, c) * inv_l - p));
            }
        }
    }
}

template <typename T, int G, int NV, bool HELD, bool ONE> static int go_mode(const DistillArgs& a, int mode, hipStream_t st) {
    constexpr int ROWS = G > 64 ? 1 : 256 / G, NT = G > 64 ? G : 256;
    const int64_t blocks = (a.rows + ROWS - 1) / ROWS;
    if (blocks * NT >= (int64_t)1 << 32) return V2VAE_ESIZE;  // a launch holds fewer threads
    const dim3 grid((unsigned)blocks);
    if (mode == DO_LOSS) hipLaunchKernelGGL((k_distill<T, G, NV, HELD, DO_LOSS, ONE>), grid, dim3(NT), 0, st, a);
    else if (mode == DO_GRAD) hipLaunchKernelGGL((k_distill<T, G, NV, HELD, DO_GRAD, ONE>), grid, dim3(NT), 0, st, a);
    else hipLaunchKernelGGL((k_distill<T, G, NV, HELD, DO_LOSS | DO_GRAD, ONE>), grid, dim3(NT), 0, st, a);
    return dense_launch_error("distillation");
}
template <typename T, int G, int NV, bool HELD> static int go(const DistillArgs& a, int mode, hipStream_t st) {
    if constexpr (G > 64) {
        if (a.k > 64) return go_mode<T, G, NV, HELD, false>(a, mode, st);
    }
    return go_mode<T, G, NV, HELD, true>(a, mode, st);
}

// The group that holds a row has a lane for every teacher entry, up to 64 of them; more are the workgroup's, which keeps them in
// LDS.  (Entries without a lane or LDS of their own, read again for every other one, took 98 us for 2 rows of 96 logits with 90
// entries and 54 for 6984 rows of 65 with 50; 16 and 16 this way.)
template <typename T> static int distill(const DistillArgs& a, int mode, hipStream_t st) {
    constexpr int E = Vec16<T>::N;
    // pieces of a row: V / E if every row starts at one, else of a row that starts anywhere
    const bool aligned = ((uintptr_t)a.z & 15) == 0 && (a.ld_z % E == 0 || a.rows == 1);
    const int64_t pieces = aligned ? (a.V + E - 1) / E : (a.V + 2 * E - 2) / E;
    // The loss alone needs no row held: many long rows stream through smaller workgroups (bf16 losses, held / streamed: 2688 x 17029 37 /
    // 24 us, 4096 x 32000 53 / 44; f16 20000 x 6000 49 / 52, therefore held, and few rows have too few workgroups this way).
    // (Rows beyond 2^22 are left to the held form, whose launch limits then refuse the same sizes for the loss as for the gradient.)
    if (mode == DO_LOSS && pieces > 1024 && pieces <= 8192 && a.rows >= 512 && a.rows < (int64_t)1 << 22)
        return go<T, 256, 4, false>(a, mode, st);
    if (pieces <= 8 && a.k <= 8) return go<T, 8, 1, true>(a, mode, st);
    if (pieces <= 16 && a.k <= 16) return go<T, 16, 1, true>(a, mode, st);
    if (pieces <= 32 && a.k <= 16) return go<T, 16, 2, true>(a, mode, st);
    if (pieces <= 64 && a.k <= 32) return go<T, 32, 2, true>(a, mode, st);
    if (pieces <= 64 && a.k <= 64) return go<T, 64, 1, true>(a, mode, st);
    if (pieces <= 256 && a.k <= 64) return go<T, 64, 4, true>(a, mode, st);
    if (pieces <= 256) return go<T, 256, 1, true>(a, mode, st);
    if (pieces <= 1024) return go<T, 256, 4, true>(a, mode, st);
    if (pieces <= 2048) return go<T, 256, 8, true>(a, mode, st);
    if (pieces <= 4096) return go<T, 512, 8, true>(a, mode, st);
    if (pieces <= 8192) return go<T, 1024, 8, true>(a, mode, st);
    return go<T, 1024, 4, false>(a, mode, st);
}

static int check_distill(const v2vae_distill* d) {
    if (!d || d->dtype < V2VAE_F32 || d->dtype > V2VAE_F16 || d->teacher_dtype < V2VAE_F32 || d->teacher_dtype > V2VAE_F16) return V2VAE_EINVAL;
    if ((d->index_bits != 32 && d->index_bits != 64) || d->reserved != 0 || d->k < 1 || d->rows < 0 || d->vocab < 1) return V2VAE_EINVAL;
    if (!(d->temperature >= 1e-4f && d->temperature <= 1e4f)) return V2VAE_EINVAL;
    if (d->ld_logits < d->vocab || d->ld_teacher < d->k || d->ld_index < d->k) return V2VAE_EINVAL;
    if (d->k > V2VAE_DISTILL_MAX_K || d->rows > ((int64_t)1 << 30) || d->vocab > ((int64_t)1 << 30)) return V2VAE_ESIZE;
    return V2VAE_OK;
}

static int run_distill(const v2vae_distill* d, const void* logits, const void* teacher, const void* index, const float* weight,
                       float* loss, float* stats, void* grad, int mode, void* stream) {
    const int rc = check_distill(d);
    if (rc != V2VAE_OK) return rc;
    if (d->rows == 0) return V2VAE_OK;
    auto bytes = [](int t) { return t == V2VAE_F32 ? 4 : 2; };
    auto off = [](const void* p, int n) { return ((uintptr_t)p % n) != 0; };
    if (!logits || !teacher || !index || off(logits, bytes(d->dtype)) || off(teacher, bytes(d->teacher_dtype)) || off(index, d->index_bits / 8))
        return V2VAE_EINVAL;
    if ((mode & DO_LOSS) && (!loss || off(loss, 4))) return V2VAE_EINVAL;
    if ((mode & DO_GRAD) && (!grad || !weight || off(grad, bytes(d->dtype)) || off(weight, 4))) return V2VAE_EINVAL;
    if (off(stats, 4) || (mode == DO_GRAD && !stats)) return V2VAE_EINVAL;
    DistillArgs a = {};
    a.z = logits;
    a.t = teacher;
    a.index = index;
    a.weight = weight;
    a.loss = loss;
    a.stats = stats;
    a.grad = grad;
    a.ld_z = d->ld_logits;
    a.ld_t = d->ld_teacher;
    a.ld_i = d->ld_index;
    a.rows = d->rows;
    a.V = (int)d->vocab;
    a.k = d->k;
    a.teacher_dtype = d->teacher_dtype;
    a.wide_index = d->index_bits == 64;
    a.T = d->temperature;
    a.inv_t = 1.f / d->temperature;
    if (d->dtype == V2VAE_F32) return distill<float>(a, mode, (hipStream_t)stream);
    if (d->dtype == V2VAE_BF16) return distill<bf16_t>(a, mode, (hipStream_t)stream);
    return distill<f16_t>(a, mode, (hipStream_t)stream);
}

}  // namespace v2vae

using namespace v2vae;

extern "C" {

int v2vae_distill_fwd(const v2vae_distill* d, const void* logits, const void* teacher, const void* index, float* loss, float* stats,
                      void* stream) {
    return run_distill(d, logits, teacher, index, nullptr, loss, stats, nullptr, DO_LOSS, stream);
}

int v2vae_distill_bwd(const v2vae_distill* d, const void* logits, const void* teacher, const void* index, const float* stats,
                      const float* weight, void* grad, void* stream) {
    return run_distill(d, logits, teacher, index, weight, nullptr, const_cast<float*>(stats), grad, DO_GRAD, stream);
}

int v2vae_distill_step(const v2vae_distill* d, const void* logits, const void* teacher, const void* index, const float* weight,
                       float* loss, void* grad, void* stream) {
    return run_distill(d, logits, teacher, index, weight, loss, nullptr, grad, DO_LOSS | DO_GRAD, stream);
}

}  // extern "C"
