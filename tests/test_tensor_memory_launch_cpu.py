"""Sources of the kernels with tensor memory: the next kernel is let in behind this one's allocation.

An allocation waits until the SM has the columns. A CTA of the next kernel that came in before it could take columns and then wait for
this kernel's end, while this one waits for the columns; neither wait has a limit."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "create_llm_by_cupy_b200" / "ops" / "csrc"


def kernels():
    for f in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", f.read_text())
        for part in re.split(r"__global__", text)[1:]:
            body = part.split("\n}\n", 1)[0]
            if re.search(r"tmem_alloc(_pair)?\(", body) and "pdl_trigger()" in body:
                yield pytest.param(body, id=f"{f.name}:{re.search(r'(\w+_kernel)', body).group(1)}")


def test_there_are_some():
    assert len(list(kernels())) >= 4


@pytest.mark.parametrize("body", list(kernels()))
def test_a_barrier_between_the_allocation_and_the_next_kernel(body):
    alloc = re.search(r"tmem_alloc(_pair)?\(", body).start()
    assert re.search(r"__syncthreads\(\)", body[alloc:body.index("pdl_trigger()")]), "the next kernel may come in before the allocation"
