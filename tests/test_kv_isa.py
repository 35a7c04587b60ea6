"""What the compiler made of the paged cache's and its attention's kernels, checked on the CPU from the gfx950 assembly as
test_isa_health.py does for the older ones: every form is there, registers do not spill beyond the few of one form, and a prompt's whole
tiles take their products in one run between two barriers."""
import re
import tempfile
from concurrent.futures import ThreadPoolExecutor

import pytest

from test_isa_health import assembly_of

FILES = ["twm_kv_cache.hip", "twm_attn_decode.hip", "twm_attn_prompt.hip"]
# e4m3 tiles are held in registers on their way to LDS, beside the sums of 128 values; two workgroups share a compute unit
SPILLS = {"13k_attn_promptILi128ELb1E": 40}   # bytes a lane


@pytest.fixture(scope="module")
def kernels():
    with tempfile.TemporaryDirectory() as d:
        with ThreadPoolExecutor(max_workers=len(FILES)) as pool:
            texts = list(pool.map(lambda f: assembly_of(f, d), FILES))
    found = {}
    for text in texts:
        for m in re.finditer(r"\n(_ZN3twm\w+):[^\n]*\n(.*?)\n\.Lfunc_end", text, re.S):
            spill = re.search(r"\.set " + re.escape(m.group(1)) + r"\.private_seg_size, (\d+)", text)
            if spill:
                found[m.group(1)] = (m.group(2), int(spill.group(1)))
    return found


def test_every_form_is_there_and_none_spills(kernels):
    for kernel, forms in (("k_kv_appendI", 2), ("k_kv_copy_pagesE", 1), ("k_attn_decodeI", 12), ("k_attn_joinI", 6), ("k_attn_promptI", 4), ("k_attn_prompt_pairsI", 6),
                          ("k_attn_prompt_joinI", 6)):
        assert sum("%d%s" % (len(kernel) - 1, kernel) in name for name in kernels) == forms, kernel
    for name, (_, scratch) in kernels.items():
        most = [b for part, b in SPILLS.items() if part in name]
        assert scratch <= (most[0] if most else 0), (name, scratch)


def test_whole_tiles_keep_their_sums_in_place(kernels):
    # scores and values of a tile of 64 tokens and 128 values: 16 products each, and no move of the sums among registers between them
    (body,) = [body for name, (body, _) in kernels.items() if "13k_attn_promptILi128ELb0E" in name]
    lines = [line.strip() for line in body.split("\n") if line.strip() and not line.strip().startswith((";", "."))]
    products = [i for i, line in enumerate(lines) if line.startswith("v_mfma")]
    assert len(products) >= 64
    run = lines[products[0]:products[31] + 1]
    assert sum(line.startswith("v_mfma") for line in run) == 32
    assert sum(line.startswith(("v_accvgpr", "scratch_")) for line in run) == 0
    assert sum(line.startswith("v_mov_b32") for line in run) <= 8
    # keys are read two steps ahead of their products
    first = [i for i, line in enumerate(lines) if line.startswith("ds_read_b128")]
    assert sum(i < products[0] for i in first) >= 4
