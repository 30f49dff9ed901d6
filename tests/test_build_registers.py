"""The build's check of the registers that kernels are built with."""
import pytest

from fold_b200 import build


def entry(name, registers):
    return (f"ptxas info    : Compiling entry function '{name}' for 'sm_100a'\n"
            f"ptxas info    : Function properties for {name}\n"
            "    48 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads\n"
            f"ptxas info    : Used {registers} registers, used 1 barriers, 48 bytes cumulative stack size\n")


def log(wide=168, narrow=168):
    return (entry("_ZN4fold1a19prefix_merge_kernelILi256E6__halfLi1EEEvNS0_12PrefixParamsEi", 56)
            + entry("_ZN4fold1a18prefix_read_kernelINS0_3CfgILi256E6__halfEEEEvNS0_12PrefixParamsE", 250)
            + entry("_ZN4fold1a18prefix_read_kernelINS0_3CfgILi128E6__halfEEEEvNS0_12PrefixParamsE", wide)
            + entry("_ZN4fold1a18prefix_read_kernelINS0_3CfgILi64E13__nv_bfloat16EEEEvNS0_12PrefixParamsE", narrow))


def test_registers_as_they_must_be():
    build.check_registers("prefix_read", log())
    build.check_registers("rope", "")


@pytest.mark.parametrize("text", [log(wide=160), log(narrow=170), entry("other", 168), ""])
def test_other_registers_fail_the_build(text):
    with pytest.raises(RuntimeError, match="prefix_read.*168"):
        build.check_registers("prefix_read", text)
