// emu_optim.h -- what mc_optim.cu and mc_optim.c use beyond emu.h and
// fake_cudart.cpp (test infrastructure only).
#pragma once

extern "C" inline __attribute__((used)) cudaError_t cudaDeviceGetAttribute(int *v, cudaDeviceAttr, int) {
    *v = 2;   // two SMs: grids that stride over their units even in small cases
    return cudaSuccess;
}
