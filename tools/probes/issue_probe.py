#!/usr/bin/env python3
"""Round 6, second probe: what ONE instruction costs a wave by encoding size, address parity and dependence - loops of 480 instructions
of one kind or a short pattern, one wave on an idle device (timing only). Behind tools/probes/chain_regs_probe.py's finding that an 8-byte
instruction at an odd word costs a clock more, and tools/align_asm.py's A / B that found the decoder 5 % SLOWER with its 4-byte VALU
instructions promoted to 8-byte ones.
    python tools/probes/issue_probe.py /tmp/issue_probe.hip && hipcc --offload-arch=gfx950 -Xclang -target-feature -Xclang -packed-fp32-ops -O2 /tmp/issue_probe.hip -o tools/probes/issue_probe.bin
"""
import sys

K = []


def add(name, desc, pattern, pad=0, n=480):
    body = (pattern * (n // len(pattern) + 1))[:n - n % len(pattern)]
    K.append((name, desc, body, len(body), pad))


E32i = ["v_mov_b32_e32 v30, v31"]
E64i = ["v_mov_b32_e64 v30, v31"]
E32d = ["v_add_u32_e32 v30, v30, v31"]
E64d = ["v_add_u32_e64 v30, v30, v31"]
V3d = ["v_add3_u32 v30, v30, v31, v31"]           # VOP3-only
SAL = ["s_add_u32 s52, s52, s53"]
SAL8 = ["s_add_u32 s52, s52, 0x12345"]
for pad in (0, 1):
    t = "odd word" if pad else "even word"
    add(f"i_e32_{pad}", f"independent 4-byte VALU (v_mov_b32_e32), loop at an {t}", E32i, pad)
    add(f"i_e64_{pad}", f"independent 8-byte VALU (v_mov_b32_e64), loop at an {t}", E64i, pad)
    add(f"d_e32_{pad}", f"dependent 4-byte VALU (v_add_u32_e32 v30, v30, v31), {t}", E32d, pad)
    add(f"d_e64_{pad}", f"dependent 8-byte VALU (v_add_u32_e64), {t}", E64d, pad)
    add(f"d_v3_{pad}", f"dependent VOP3-only (v_add3_u32), {t}", V3d, pad)
    add(f"s_4_{pad}", f"dependent 4-byte SALU (s_add_u32), {t}", SAL, pad)
    add(f"s_8_{pad}", f"dependent 8-byte SALU (s_add_u32 with a literal), {t}", SAL8, pad)
    add(f"d_448_{pad}", f"dependent e32, e32, e64 (the e64 {'mis' if pad else ''}aligned), {t}", E32d + E32d + E64d, pad)
    add(f"d_484_{pad}", f"dependent e32, e64, e32 (the e64 {'' if pad else 'mis'}aligned), {t}", E32d + E64d + E32d, pad)
    add(f"d_48_{pad}", f"dependent e32, e64 alternating (every e64 {'aligned' if pad else 'misaligned'}), {t}", E32d + E64d, pad)
    add(f"d_4888_{pad}", f"dependent e32 then three e64 (parity flips every 4 instructions), {t}", E32d + E64d * 3, pad)
    add(f"i_48_{pad}", f"independent e32, e64 alternating, {t}", E32i + E64i, pad)
    add(f"i_4888_{pad}", f"independent e32 then three e64, {t}", E32i + E64i * 3, pad)
    add(f"d_f64_{pad}", f"dependent v_fma_f64, {t}", ["v_fma_f64 v[32:33], v[32:33], v[34:35], v[34:35]"], pad)
    add(f"d_fmac32_{pad}", f"dependent v_fmac_f64_e32 (4 bytes), {t}", ["v_fmac_f64_e32 v[32:33], v[34:35], v[34:35]"], pad)
    add(f"d_ds_{pad}", f"independent ds_read_b32 (8 bytes), {t}", ["ds_read_b32 v36, v37"], pad, 96)


def emit(out):
    f = open(out, "w")
    f.write("// generated by tools/probes/issue_probe.py - timing only\n#include <hip/hip_runtime.h>\n#include <stdio.h>\n#include <stdint.h>\n#include <string.h>\n")
    clob = ", ".join(f'"v{i}"' for i in range(28, 40)) + ', "s52", "s53", "s60", "s62", "s63", "s64", "s65", "scc", "vcc", "memory"'
    pro = ["v_mov_b32 v30, 1", "v_mov_b32 v31, 3", "v_mov_b32 v32, 0", "v_mov_b32 v33, 0x3ff00000", "v_mov_b32 v34, 0", "v_mov_b32 v35, 0x3ff00000", "v_mov_b32 v37, 0", "s_mov_b32 s52, 0", "s_mov_b32 s53, 1",
           "s_mov_b32 s60, %[it]", "s_nop 4", "s_memtime s[62:63]", "s_waitcnt lgkmcnt(0)"]
    epi = ["s_sub_u32 s60, s60, 1", "s_cmp_lg_u32 s60, 0", "s_cbranch_scc1 1b", "s_waitcnt vmcnt(0) lgkmcnt(0)", "s_memtime s[64:65]", "s_waitcnt lgkmcnt(0)", "s_sub_u32 %[clk], s64, s62"]
    for name, desc, body, n, pad in K:
        f.write(f"__global__ void __launch_bounds__(64) k_{name} (uint64_t *out, uint32_t iters)\n{{\n    uint32_t clocks;\n    __shared__ uint32_t lds[64];\n    if (iters == 0xffffffffu) lds[threadIdx.x] = 1;\n    asm volatile (\n")
        for ln in pro + [".p2align 6"] + ["s_nop 0"] * pad + ["1:"] + body + epi:
            f.write(f'        "{ln}\\n\\t"\n')
        f.write(f'        : [clk] "=s" (clocks) : [it] "s" (iters) : {clob});\n    if (!threadIdx.x) out[0] = clocks;\n    if (iters == 0xffffffffu) out[1] = lds[5];\n}}\n')
    f.write("struct P { const char *name, *desc; void (*k) (uint64_t *, uint32_t); uint32_t n; } Ps[] = {\n")
    for name, desc, body, n, pad in K:
        f.write(f'    {{ "{name}", "{desc}", k_{name}, {n} }},\n')
    f.write("};\n")
    f.write(r"""
int main (int argc, char **argv)
{
    uint64_t *d, h[2];
    if (hipMalloc (&d, 16) != hipSuccess) { printf ("no device\n"); return 1; }
    for (unsigned i = 0; i < sizeof (Ps) / sizeof (Ps[0]); i++) {
        if (argc > 1 && !strstr (Ps[i].name, argv[1])) continue;
        const uint32_t iters = 2000000u / Ps[i].n;
        double best = 1e30;
        for (int rep = 0; rep < 3; rep++) {
            hipLaunchKernelGGL (Ps[i].k, dim3 (1), dim3 (64), 0, 0, d, iters);
            if (hipDeviceSynchronize () != hipSuccess) { printf ("%s: failed\n", Ps[i].name); return 1; }
            (void)hipMemcpy (h, d, 16, hipMemcpyDeviceToHost);
            const double c = (double)(uint32_t)h[0] / ((double)iters * Ps[i].n);
            if (c < best) best = c;
        }
        printf ("%-14s %7.3f clocks per instruction   %s\n", Ps[i].name, best, Ps[i].desc);
        fflush (stdout);
    }
    return 0;
}
""")
    f.close()


if __name__ == "__main__":
    emit(sys.argv[1])
    print(len(K), "kernels")
