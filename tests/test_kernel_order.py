"""What the sources have to hold for kernels that run one behind the other: tensor memory is taken in front of the signal that lets the next
kernel's CTAs in.  Behind it, a CTA of the next kernel on the same SM could hold the tensor memory that this one waits for, while it waits for this
kernel to end.  Read here, since the other order shows in nothing but a hang."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse-winograd-cnn_b200", "csrc")
TAKES = re.compile(r"\btmem_alloc\(|tcgen05\.alloc\.")
LETS_IN = re.compile(r"\b(wait_for_previous_kernel|after_previous_kernel|let_next_kernel_in)\(|griddepcontrol\.launch_dependents")


def kernels(text):
    """(name, body) of the kernels of a source"""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"__global__", text):
        at = text.index("{", m.end())
        name = re.findall(r"(\w+)\s*\(", text[m.end():at])
        depth, end = 1, at + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield [n for n in name if n not in ("__launch_bounds__", "__cluster_dims__")][0], text[at:end]


def early(text):
    """Kernels that let the next one in before they have their tensor memory"""
    out = []
    for name, body in kernels(text):
        takes, lets = TAKES.search(body), LETS_IN.search(body)
        if takes and lets and lets.start() < takes.start():
            out.append(name)
    return out


def test_tensor_memory_is_taken_before_the_next_kernel_comes_in():
    found = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        text = open(path).read()
        assert early(text) == [], os.path.basename(path)
        found += sum(bool(TAKES.search(body)) for _, body in kernels(text))
    assert found >= 8


def test_the_reading_sees_the_other_order():
    planted = """
    template <int N> __global__ void __launch_bounds__(64, 1) one_kernel(int a) { if (a) { wait_for_previous_kernel(4); } tmem_alloc(0, 32); }
    __global__ void two_kernel(int a) { tmem_alloc(0, 32); after_previous_kernel(a); }
    """
    assert early(planted) == ["one_kernel"]
