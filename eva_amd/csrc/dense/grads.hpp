// Parameters of the gradients' kernels.
#pragma once
#include "linear.hpp"

namespace evamx_dense {

struct ActGradParams {
    const uint16_t* grad;
    size_t grad_stride;
    const float* pre;
    uint16_t* out;               // [rows][out_stride]
    size_t out_stride;
    Groups g;
    int n_out, act;
    float limit;
};

struct WeightGradParams {
    const uint16_t* x;
    const uint16_t* d;
    size_t x_stride, d_stride;
    uint16_t* out;               // [experts][n_out][n_in]
    Groups g;
    bool stream;                 // out is more than the last-level cache holds
    int n_in, n_out;
    int x_cols, d_cols;          // values in a row of x and d: multiples of 8, zeros behind the last
    float* part;                 // [splits][n_out][n_in] (one expert)
    Plan plan;
};

struct ColumnSumParams {
    const uint16_t* d;
    size_t d_stride;
    uint16_t* out;               // [experts][n_out]
    Groups g;
    int n_out;
    float* part;                 // [experts][parts][n_out]
    int parts;
};

int launch_act_grad(const ActGradParams& p, int dtype, hipStream_t s);
int launch_weight_grad(const WeightGradParams& p, int dtype, hipStream_t s);
int launch_column_sums(const ColumnSumParams& p, int dtype, hipStream_t s);

}  // namespace evamx_dense
