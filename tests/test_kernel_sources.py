"""What the kernels' sources promise beyond what a compiler checks: alignment of shared arrays that are used 16 bytes at a time, and no
helper without a caller."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "610sample_b200", "csrc")


def sources():
    found = {}
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            found[name] = re.sub(r"//[^\n]*", "", f.read())
    return found


def test_shared_arrays_used_by_16_bytes_are_aligned():
    for name, text in sources().items():
        for kernel in text.split("__global__"):
            for decl in re.findall(r"__shared__\s+([^;]*);", kernel):
                if "__align__" in decl or re.match(r"(u?int4|float4|PackedTile)\b", decl):
                    continue
                for array in re.findall(r"\b(\w+)\s*\[", decl):
                    wide = re.search(r"reinterpret_cast<(const )?(float4|uint4|int4)\s*\*>\(&?%s\b" % array, kernel)
                    assert wide is None, f"{name}: {array} is read or written by 16 bytes, and declared with less: {decl}"


def test_device_helpers_have_callers():
    texts = sources()
    everything = "\n".join(texts.values())
    for name, text in texts.items():
        for helper in re.findall(r"__device__ __forceinline__ [\w:<>, \t*&]*?\b(\w+)\(", text):
            uses = len(re.findall(r"\b%s\b" % helper, everything))
            definitions = len(re.findall(r"__device__ __forceinline__ [\w:<>, \t*&]*?\b%s(?:<\w+>)?\(" % helper, everything))
            assert uses > definitions, f"{name}: {helper} has no caller"
