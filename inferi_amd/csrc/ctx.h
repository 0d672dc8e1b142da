// The context behind the C ABI: one device, one stream, the loaded kernels.
#pragma once
#include <hip/hip_runtime_api.h>

#include <cstdarg>
#include <cstdio>
#include <map>
#include <string>

#include "../../include/inferi_hip.h"
#include "kargs.h"

struct ifr_ctx {
    int device = 0;
    hipStream_t stream = nullptr;
    hipModule_t module = nullptr;
    hipModule_t paged_module = nullptr; // kernels named paged_* (inferi_paged.hsaco)
    std::map<std::string, hipFunction_t> fns;
    // kernels of ifr_matmul_quant's f32 input by type id: rows of one K step
    // and longer ones (looked up at a type's first call)
    struct PlainXf {
        bool known = false;
        hipFunction_t one = nullptr, loop = nullptr;
    } plain_xf[16];
    ifr::StepCtl *ctl_host = nullptr; // pinned: a state's control block read back
    std::string err;
    char dev_name[256] = {0};
    int n_cu = 0;
    hipEvent_t events[16] = {};
    // scratch for the op-level attention and argmax
    void *scratch = nullptr;
    size_t scratch_bytes = 0;
    // quantized activation of the op-level GEMV
    void *xq_scratch = nullptr;
    size_t xq_scratch_bytes = 0;
    // tuning: cap on GEMV workgroups (0 = one per row tile)
    uint32_t gemv_max_grid = 0;
    uint32_t gemv_waves = 0; // integer-path waves per workgroup (0: by shape)
    // GEMV arithmetic: 0 = x as 16-bit fixed point with int8 dot products,
    // 1 = exact fp32 x and FMAs
    int gemv_exact = 0;
    // one-item GEMV forms in use: bit 0 resid with one K step (O), bit 1
    // resid with K-slices (down), bit 2 gateup, bit 3 gateup as 16 waves of
    // two rows (else 8 waves of four), bit 4 the output head, bit 5 gateup
    // with h in f32 and the down GEMV quantizing it, bit 6 the Q6_K head in
    // 256-VGPR workgroups, bit 7 gateup with four rows per wave, bit 8 plain
    // and qkv with four rows per wave (default: bits 0, 5, 6 and 7)
    int gemv_grp = 225;
    // prompt tokens per prefill pass (0: PF_CHUNK), read at a state's first prefill
    uint32_t pf_chunk = 0;
    // this device's fixed scratch of ifr_matmul_quant_noalloc (noalloc.hip)
    void *noalloc_scratch = nullptr;
    // prefill GEMM tiles: 0 = by shape (pf_small_form), 128 or 256 to force
    // one (option pf_tile)
    uint32_t pf_tile = 0;
    // Q4_K products on 256 x 256 tiles in the warp-specialized form (option
    // pf_ws, default on; 0 = the eight-wave form; device/pf_gemm.h
    // pf_gemm_ws_body)
    int pf_ws = 1;
    // the Q/K/V product's epilogue applies RoPE and stores k, v to the cache
    // (not in the eight-wave form; pairs (2i, 2i + 1)) instead of pf_rope_kv_k
    // (option pf_rope_fuse, default on)
    int pf_rope_fuse = 1;
    // bumped by every option change: a captured decode step is captured
    // again when it differs
    uint64_t opt_gen = 0;

    ifr_status fail(ifr_status st, const char *fmt, ...) {
        char buf[1024];
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(buf, sizeof buf, fmt, ap);
        va_end(ap);
        err = buf;
        return st;
    }
    ifr_status hip(hipError_t e, const char *what) {
        if (e == hipSuccess) return IFR_OK;
        return fail(e == hipErrorOutOfMemory ? IFR_ENOMEM : IFR_EHIP, "%s: %s", what, hipGetErrorString(e));
    }
    hipFunction_t fn(const std::string &name) {
        auto it = fns.find(name);
        if (it != fns.end()) return it->second;
        hipFunction_t f = nullptr;
        // asked only for kernels that the code object has: a failed look-up
        // would set the thread's last HIP error, and clearing that one would
        // take away an error that the program itself left there
        hipModule_t from = name.compare(0, 6, "paged_") ? module : paged_module;
        if (from && hipModuleGetFunction(&f, from, name.c_str()) != hipSuccess) f = nullptr;
        fns[name] = f;
        return f;
    }
    template <class A>
    ifr_status launch(const std::string &name, dim3 grid, dim3 block, uint32_t shmem, const A &args) {
        hipFunction_t f = fn(name);
        if (!f) return fail(IFR_EUNSUPPORTED, "kernel %s not in the code object", name.c_str());
        return launch_fn(f, name.c_str(), grid, block, shmem, args);
    }
    template <class A>
    ifr_status launch_fn(hipFunction_t f, const char *name, dim3 grid, dim3 block, uint32_t shmem, const A &args) {
        // every kernel takes one struct argument: kernelParams[0] points at it
        void *params[] = {const_cast<A *>(&args)};
        return hip(hipModuleLaunchKernel(f, grid.x, grid.y, grid.z, block.x, block.y, block.z, shmem, stream, params,
                                         nullptr),
                   name);
    }
    ifr_status ensure_xq_scratch(size_t bytes) {
        if (bytes <= xq_scratch_bytes) return IFR_OK;
        if (xq_scratch) {
            hipStreamSynchronize(stream);
            hipFree(xq_scratch);
            xq_scratch = nullptr;
            xq_scratch_bytes = 0;
        }
        ifr_status st = hip(hipMalloc(&xq_scratch, bytes), "hipMalloc(xq scratch)");
        if (st) return st;
        xq_scratch_bytes = bytes;
        return IFR_OK;
    }
    ifr_status ensure_scratch(size_t bytes) {
        if (bytes <= scratch_bytes) return IFR_OK;
        if (scratch) {
            hipStreamSynchronize(stream);
            hipFree(scratch);
            scratch = nullptr;
            scratch_bytes = 0;
        }
        ifr_status st = hip(hipMalloc(&scratch, bytes), "hipMalloc(scratch)");
        if (st) return st;
        scratch_bytes = bytes;
        return IFR_OK;
    }
};
