"""Compile-level guards of the MXFP4 and logit-control kernels: no scratch memory (a reload waits, in order, behind the transfers on their way), no packed
fp32 instructions, at most 256 registers (two waves per SIMD), and transfers to LDS whose waits leave some of them on their way.  No GPU needed."""
import re

from test_isa_regressions_cpu import compile_to_asm, kernel_bodies

FLAGS = ("-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops")


def test_operator_kernels(tmp_path):
    for source, stems in (("mxfp4", ("mx_quantize_kernel", "mx_rows_kernel", "mx_tile_kernel")), ("logits", ("logit_controls_kernel",))):
        asm, usage = compile_to_asm(source, tmp_path, FLAGS)
        assert not re.search(r"v_pk_(add|mul|fma)_f32", asm)
        for stem in stems:
            bodies = list(kernel_bodies(asm, stem))
            assert bodies
            for name, body in bodies:
                assert usage[name]["scratch"] == 0 and usage[name]["spill"] == 0 and usage[name]["vgpr"] <= 256, (name, usage[name])
                if stem == "mx_tile_kernel":
                    assert "global_load_lds_dwordx4" in body
                    deeper_than_two = not re.search(r"ILb1ELi1E", name)  # the large 4-bit tile has room for two stages
                    assert bool(re.search(r"s_waitcnt vmcnt\((?!0\))\d+\)", body)) or not deeper_than_two, name
