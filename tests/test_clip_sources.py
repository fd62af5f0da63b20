"""What the clipping kernels' source has to keep: no order of execution on one GPU shows the difference."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse_ads_baselines_b200", "csrc",
                      "tbe_grad_clip.cu")


def _definitions(text):
    """name -> body of the functions and structs at the outer level."""
    text = re.sub(r"//.*|__launch_bounds__\([^)]*\)|__grid_constant__", "", text)
    found = {}
    for m in re.finditer(r"^(?:struct (\w+) \{|(?:template <[^\n]*>\n)?__(?:device|global)__[^;{]*?\b(\w+)\([^;{]*\{)(.*?)^\}",
                         text, flags=re.M | re.S):
        name, body = m.group(1) or m.group(2), m.group(3)
        found[name] = found.get(name, "") + body
    return found


def test_a_kernel_that_scales_in_place_has_no_read_only_loads():
    """PTX allows ld.global.nc only where nothing writes the memory while the kernel runs; the one-kernel form sums
    and scales the same tensors."""
    defs = _definitions(open(SOURCE).read())
    assert "grad_clip_small_kernel" in defs and "piece_scale" in defs["grad_clip_small_kernel"]
    reached, todo = set(), ["grad_clip_small_kernel"]
    while todo:
        name = todo.pop()
        if name not in reached:
            reached.add(name)
            todo += [d for d in defs if re.search(r"\b%s\b" % d, defs[name])]
    assert {"piece_squares", "chunk_squares", "sum_squares", "scale_chunk"} <= reached
    for name in sorted(reached):
        bad = re.findall(r"\bld_stream\w*|\b__ldg\w*|\bld\.global\.nc\S*", defs[name])
        assert not bad, "%s, which grad_clip_small_kernel reaches, loads as read-only: %s" % (name, bad)
