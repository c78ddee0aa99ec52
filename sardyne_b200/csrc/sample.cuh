// Launcher of the sampling kernel (sample.cu), asynchronous on stream s.
#pragma once
#include "common.cuh"
#include "sardyne_b200.h"

namespace sdy {

// One row's parameters and uniform number, as sdy_sample_args names them.
struct SampleWords {
    float temperature;
    int32_t top_k;
    float top_p, min_p, u;
};

constexpr int SAMPLE_MAX_VOCAB = 400000;
void sample_rows(const sdy_sample_args &a, cudaStream_t s);  // arguments as sdy_sample_dev has checked them

}  // namespace sdy
