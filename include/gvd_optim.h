/*
 * gvd_optim.h -- C-ABI of the optimizer step over many tensors at once (csrc/adamw.hip).
 *
 * Plain C: raw DEVICE pointers, sizes, hipStream_t as void*.  Every function returns 0 on success or a negative code
 * (gvd_optim_last_error() has the message, per thread).  Nothing is allocated, kept or synchronised; every launch is on `stream`.
 */
#ifndef GVD_OPTIM_H_INCLUDED
#define GVD_OPTIM_H_INCLUDED

#ifdef __cplusplus
extern "C" {
#endif

/* Elements that share one scale where moments are held in 8 bits. */
#define GVD_ADAMW_BLOCK 256
/* Elements of a tensor at most. */
#define GVD_ADAMW_MOST (1LL << 34)

/* One tensor of a step.  All arrays hold n elements in the same memory order, dense; no two arrays of one call overlap.
 * state_bits 32: exp_avg, exp_avg_sq are float[n]; the scale pointers are not read.
 * state_bits 8:  exp_avg and exp_avg_sq are OCP e4m3 bytes [n]: element i of the first moment is exp_avg[i] * exp_avg_scale[i / 256], and the
 *                ROOT of the second moment is exp_avg_sq[i] * exp_avg_sq_scale[i / 256] (scales: float[(n + 255) / 256]). */
typedef struct gvd_adamw_tensor {
    void* param;
    const void* grad;
    void* exp_avg;
    void* exp_avg_sq;
    float* exp_avg_scale;
    float* exp_avg_sq_scale;
    long long n;
    float step_size;      /* lr / (1 - beta1^t) */
    float root_factor;    /* 1 / sqrt(1 - beta2^t) */
    float keep;           /* 1 - lr * weight_decay */
    unsigned key;         /* of the stochastic rounding: gvd_adamw_key(seed, tensor, t); read with state_bits 8 only */
} gvd_adamw_tensor;

/* One AdamW step over `count` tensors whose parameters and gradients have the type param_type (0 float, 1 fp16, 2 bf16):
 *     m' = m + (1 - beta1) (g - m),   v' = beta2 v + (1 - beta2) g^2
 *     p' = keep p - step_size m' / (root_factor sqrt(v') + eps)
 * in 32 bits, each result rounded once.  scalars: NULL, or a device array of 4 words a tensor (step_size, root_factor, keep, key) that
 * gvd_adamw_scalars wrote; it then takes the place of those members. */
int gvd_adamw_step(const gvd_adamw_tensor* tensors, int count, int param_type, int state_bits, double beta1, double beta2, double eps,
                   const void* scalars, void* stream);

/* The scalars of a step that counts on the device (a step inside a captured graph): for each tensor *step += 1, and scalars[4 i ..] are made
 * from the new count.  steps: device float each; lrs: device float each, or NULL for the host's lr; tensor_ids: the tensor's number in the hash. */
int gvd_adamw_scalars(float* const* steps, const float* const* lrs, const double* lr, const double* weight_decay, const unsigned* tensor_ids,
                      int count, double beta1, double beta2, unsigned seed, void* scalars, void* stream);

/* The 32-bit key of (seed, tensor, step) that the stochastic rounding's hash starts from. */
unsigned gvd_adamw_key(unsigned seed, unsigned tensor, unsigned step);

const char* gvd_optim_last_error(void);

#ifdef __cplusplus
}
#endif
#endif
