"""The build notices a register allotment that the many-row attention could not be launched with."""
import pytest

from vault_b200 import build

ENTRY = "ptxas info    : Compiling entry function '_ZN3v3g12k_kv_prefillI{}Li64EEEvNS_10KvAttnArgsEi' for 'sm_100a'\n"
OTHER = """ptxas info    : Compiling entry function '_ZN3v3g11k_kv_appendIfLi64ELb1EEEvNS_10AppendArgsE' for 'sm_100a'
ptxas info    : Function properties for _ZN3v3g11k_kv_appendIfLi64ELb1EEEvNS_10AppendArgsE
    8 bytes stack frame, 4 bytes spill stores, 4 bytes spill loads
ptxas info    : Used 72 registers, used 1 barriers, 4096 bytes smem
"""


def _log(*registers):
    return OTHER + "".join(ENTRY.format(f"6__half{i}") + f"ptxas info    : Used {n} registers, used 16 barriers\n"
                           for i, n in enumerate(registers)) + OTHER


def test_the_number_that_the_warps_shares_add_up_to():
    build.check_registers(_log(128, 128, 128, 128))


@pytest.mark.parametrize("registers", [(120,), (128, 120), (168, 128), ()])
def test_others_are_refused(registers):
    with pytest.raises(RuntimeError, match="k_kv_prefill"):
        build.check_registers(_log(*registers))
