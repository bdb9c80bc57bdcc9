"""Rules of the programming model that the head operators' kernels have to keep and that no run can show to be kept: read from
the sources."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
KERNELS = os.path.join(ROOT, "rocal_b200", "csrc", "kernels")


def _body(file, name):
    """The body of function `name`, comments taken out."""
    with open(os.path.join(KERNELS, file)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    at = text.index("{", re.search(r"\s%s\((?=[^;]*\{)" % name, text).start())
    depth = 0
    for end in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        if depth == 0:
            return text[at:end + 1]
    raise AssertionError(name)


@pytest.mark.parametrize("file,kernel,remote", [("grad_clip.cu", "clip_few_kernel", "st.shared::cluster"),
                                                ("gemm.cuh", "gemm_kernel", "tc::map_to_rank")])
def test_clusters_meet_before_they_touch_each_other(file, kernel, remote):
    """A block's shared memory may be touched by another one only once it is known to have started: a cluster barrier lies
    before the first access, and another behind the last one, so that no block has left by then."""
    body = _body(file, kernel)
    barriers = [m.start() for m in re.finditer(r"tc::cluster_(sync|wait)\(\)", body)]
    accesses = [m.start() for m in re.finditer(re.escape(remote), body)]
    assert accesses and barriers and barriers[0] < accesses[0] and accesses[-1] < barriers[-1], (kernel, barriers, accesses)
    assert body.count("tc::cluster_arrive()") == body.count("tc::cluster_wait()")


def test_what_a_kernel_writes_it_reads_coherently():
    """__ldg is for data that no one writes while the kernel runs. The clipping of few elements reads its gradients and writes them
    in place in one launch: the sum of squares that it makes asks for plain loads, the loads of the norm's own launch may be __ldg."""
    few, norm = _body("grad_clip.cu", "clip_few_kernel"), _body("grad_clip.cu", "clip_norm_kernel")
    assert "square_piece<false>" in few and "square_piece<true>" in norm and "__ldg" not in few
    assert "__ldg" not in _body("grad_clip.cu", "square_sum") and "square_sum<STAYS>" in _body("grad_clip.cu", "square_piece")
    for name in ("scale_vectors", "scale_chunk", "load_words"):          # these write the same tensors
        assert "__ldg" not in _body("grad_clip.cu", name)


@pytest.mark.parametrize("waits_for", [r"full\(s\)", "drained"])
@pytest.mark.parametrize("file,kernel", [("gemm.cuh", "gemm_kernel"), ("narrow_loss.cuh", "ce_narrow_kernel")])
def test_copies_and_products_in_flight_are_waited_for(file, kernel, waits_for):
    """A block must not end while a copy into its shared memory is on its way, or a product that it has issued. Where another warp gives up
    on a wait, the warp that issues the copies (the products) may have issued its last one already: its own wait for them must not
    depend on whether it has been told."""
    body = _body(file, kernel)
    loops = [m.start() for m in re.finditer(r"tc::bar_drain\(" + waits_for, body)]
    assert loops
    at, depth, conditions = loops[0], 0, []
    for i in range(at, body.index("tc::elect_one()"), -1):      # the blocks that the wait lies in
        depth += {"}": 1, "{": -1}.get(body[i], 0)
        if body[i] == "{" and depth < 0:
            conditions.append(re.split(r"[;{}]", body[:i])[-1] if "for" not in body[max(0, i - 80):i] else "for")
            depth = 0
    assert conditions and not any(re.search(r"\bok\b|gave_up", c) for c in conditions), conditions
