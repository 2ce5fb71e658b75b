"""Attention behind a shared prefix where some sequences are long enough to read it by themselves and others read it together, with
more than 64 sequences, and prompts of head dimensions between the kernels' widths."""
import numpy as np
import pytest

from paged_reference import Case
from test_gpu_paged_attn import Device, check

pytestmark = pytest.mark.gpu

# new and own tokens; of 4 query heads a key head, sequences of more than 64 new tokens read the prefix by themselves
LONG_FIRST = ((200, 210), (1, 4), (3, 9), (130, 131), (1, 1), (2, 5), (1, 7))
LONG_AMID = ((2, 9), (1, 40), (300, 301), (1, 2), (0, 3), (60, 90), (65, 70), (1, 1), (4, 4), (3, 300), (1, 8))
MIXED = {
    "first": dict(lens=LONG_FIRST, prefix=300, D=64),
    "first_d128": dict(lens=LONG_FIRST, prefix=300, D=128, dtype="bf16", order="lh"),
    "amid": dict(lens=LONG_AMID, prefix=333, D=128, page=24),
    "amid_d64": dict(lens=LONG_AMID, prefix=64, D=64, dtype="bf16"),
    "window_slopes": dict(lens=LONG_FIRST, prefix=300, D=64, window=150, slopes=True),
    "window_amid": dict(lens=LONG_AMID, prefix=500, D=128, window=333, slopes=True, cap=9.0),
    "slopes": dict(lens=LONG_AMID, prefix=300, D=64, slopes=True),
    "all_keys": dict(lens=LONG_FIRST, prefix=129, D=64, causal=False),
    "more_new_than_cached": dict(lens=((200, 150), (5, 3), (1, 0), (2, 2), (1, 9), (3, 1), (1, 1)), prefix=200, D=64),
    "gap_and_tail": dict(lens=LONG_AMID, prefix=300, D=128, gap=9, tail=200),
}


@pytest.mark.parametrize("name", list(MIXED))
def test_sequences_that_read_the_prefix_alone_beside_others(gpu, name):
    case = Case(seed=sum(map(ord, name)), Hq=8, Hkv=2, **MIXED[name])
    check(gpu, case, 0)
    gpu.kernel_log_clear()
    Device(gpu, case).launch()
    log = gpu.kernel_log()
    gpu.synchronize()
    # the long sequences', the prefix of the others, their own keys, both joined
    assert log.count("paged_tile_kernel") == 2 and "paged_rows_kernel" in log and "paged_join_kernel" in log, log


MANY = {
    "decode_70": dict(lens=tuple((1, 1 + (i * 7) % 50) for i in range(70)), prefix=200, Hq=8, Hkv=2, D=64),
    "decode_150": dict(lens=tuple((1 if i % 5 else 2, 2 + (i * 7) % 190) for i in range(150)), prefix=700, Hq=4, Hkv=2, D=128,
                       dtype="bf16"),
    "window_130": dict(lens=tuple((i % 3, 2 + (i * 7) % 50) for i in range(130)), prefix=300, window=170, slopes=True, Hq=8, Hkv=2,
                       D=64),
    "long_among_100": dict(lens=tuple((90 if i in (3, 66, 99) else 1, 90 + i % 9) for i in range(100)), prefix=260, Hq=8, Hkv=2,
                           D=64),
    "without_prefix_200": dict(lens=tuple((80 if i % 67 == 0 else i % 2, 80 + (i * 7) % 90) for i in range(200)), Hq=8, Hkv=2,
                               D=64),
}


@pytest.mark.parametrize("name", list(MANY))
@pytest.mark.parametrize("kernel", [0, 2, 3, 4])
def test_more_sequences_than_lanes(gpu, kernel, name):
    """Sequences past the 64th are not in the lanes' registers, and their shares lie behind those of earlier ones."""
    check(gpu, Case(seed=sum(map(ord, name)), **MANY[name]), kernel)


@pytest.mark.parametrize("D", [8, 24, 72, 80, 96, 104, 120])
@pytest.mark.parametrize("kernel", [0, 2, 3, 4])
def test_prompts_between_the_kernels_widths(gpu, kernel, D):
    """Several tiles and blocks at head dimensions that fill 64 or 128 columns in part."""
    dtype = "f16" if D % 16 else "bf16"
    check(gpu, Case(lens=((150, 150), (70, 333), (1, 200), (300, 301)), Hq=4, Hkv=2, D=D, dtype=dtype, seed=D,
                    order="lh" if D == 80 else "hl", window=100 if D == 104 else 0, cap=8.0 if D == 72 else 0.0), kernel)


@pytest.mark.parametrize("prefix", [0, 150])
def test_capped_prompts_between_the_kernels_widths(gpu, prefix):
    check(gpu, Case(lens=((150, 150), (70, 333), (300, 301)), Hq=4, Hkv=2, D=96, cap=3.0, q_size=3.0, slopes=True, prefix=prefix,
                    seed=51), 0)
