"""A kernel that takes tensor memory after it has waited for the kernels before it lets the next one start only when it has what it wants: a block of the next kernel that came first
would hold columns while it waits for this kernel, which would wait for them.  (Read from the source: on a device the two orders differ in nothing but in when they fail.)"""
from __future__ import annotations

import re
from pathlib import Path

SOURCES = Path(__file__).resolve().parent.parent / "hyperion_b200" / "csrc"


def test_tiles_behind_shared_positions():
    text = (SOURCES / "attention_shared_tiles.cu").read_text()
    kernel = text[text.index("attention_shared_kernel("): text.index("// Operands of 8-bit records")]
    waited, taken, met, started = (kernel.index(what) for what in ("wait_for_previous_kernels();", "tcgen05.alloc", "__syncthreads();\n    // Only now", "let_next_kernel_start();"))
    assert waited < taken < met < started and kernel.count("let_next_kernel_start();") == 1


def test_prompt_tiles():
    """These let the next kernel start at once, so none of its blocks may fit beside one of theirs: 228 KB an SM, one of them each block's own."""
    text, products = ((SOURCES / name).read_text() for name in ("attention_tcgen05.cu", "gemm_tcgen05.cu"))
    least = int(re.search(r"SMEM_BYTES = SMEM_USED > (\d+) \* 1024", text).group(1))
    ring = int(re.search(r"SHALLOW = \((\d+) \* 1024\) / STAGE_BYTES", products).group(1)) * 1024
    smallest = min(ring // stage * stage for stage in (128 * 128 + columns * 128 for columns in (16, 32, 64, 128, 256))) + 1024 + 256
    assert least * 1024 + 1024 + smallest + 1024 > 228 * 1024
