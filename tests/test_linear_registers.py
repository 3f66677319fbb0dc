"""No kernel of the bf16 products keeps a vector register in memory: 256 x 256 tiles have
none to spare, and a compiler that spills there would put memory into their loops."""
import device_code as dc


def test_linear_kernels_keep_their_registers(q38m, tmp_path):
    kernels = {name: r for path in dc.code_objects(q38m.LIB_PATH, tmp_path) for name, r in dc.resources(path).items()
               if any(part in name for part in ("linear_", "activation_backward", "bias_sum", "bias_join"))}
    assert len([name for name in kernels if "linear_tile_kernel" in name]) >= 50
    assert len([name for name in kernels if "linear_few_kernel" in name]) >= 10
    spilled = {name: (r["vgpr_spill_count"], r["private_segment_fixed_size"]) for name, r in kernels.items()
               if r["vgpr_spill_count"] or r["private_segment_fixed_size"]}
    assert not spilled, spilled
