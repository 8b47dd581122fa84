// Single translation unit of the shared library (the kernels share one
// device error word without relocatable device code).
#include "ffn_decode.hip"
#include "route.hip"
#include "grouped.hip"
#include "stack_decode.hip"
#include "rows.hip"
#include "linear_fp8.hip"
#include "attn.hip"
#include "capi.hip"
#include "capi_layer.hip"
#include "engine.hip"
#include "policy.cpp"
