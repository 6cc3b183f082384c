"""The cache operators' kernels, as compiled: none spills to memory, and all fit
the CU's LDS."""

import re

# dims 64, 128, 256 and 768, three types: attention over a cache by few and by
# many rows (in 32 bits many only at 128), with a prefix that goes three ways.
ATTEND = 4 * 2 * 2 + 4 + 1
PREFIX = 4 * 2 * 3 + 4 + 2


def _bodies(device_asm):
    return {m[1]: m[2] for (_, library), asm in device_asm.items() if library == "kernels.so"
            for m in re.finditer(r"^(_Z\w+):.*?\n(.*?)^\.Lfunc_end", asm, re.S | re.M)}


def test_every_form_is_there_once(device_asm):
    names = [n for n in _bodies(device_asm) if "5cache" in n]
    assert sum("cache_attend_kernel" in n for n in names) == ATTEND
    assert sum("cache_prefix_kernel" in n for n in names) == PREFIX
    assert sum("cache_merge_kernel" in n for n in names) == 12 * 2
    assert sum("rope_kernel" in n for n in names) == 3 * 2 * 2
    assert sum("cache_append_kernel" in n for n in names) == 3 * 2 * 2


def test_nothing_is_spilled_to_memory(device_asm):
    for name, body in _bodies(device_asm).items():
        if "5cache" in name:
            assert not re.search(r"\bscratch_(load|store)", body), name


def test_attention_fits_lds(device_asm):
    sizes = {}
    for asm in device_asm.values():
        for m in re.finditer(r"group_segment_fixed_size: *(\d+).*?\.name: *(_Z\w+)", asm, re.S):
            if "5cache" in m[2]:
                sizes[m[2]] = int(m[1])
    assert sizes and max(sizes.values()) <= 160 * 1024
