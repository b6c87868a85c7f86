"""Rules of the CUDA sources that no compiler checks."""
import re
from pathlib import Path

import lset_b200

CSRC = Path(lset_b200.__file__).parent / "csrc"
TEXTS = {p: p.read_text() for p in sorted(CSRC.rglob("*.cu*")) if "_build" not in p.parts}


def _functions(text):
    """Texts of the functions of a file, each from the line after the last closing brace in column
    zero to its own."""
    return re.split(r"\n}[^\n]*\n", text)


def _kernel_body(name):
    for text in TEXTS.values():
        for fn in _functions(text):
            if re.search(r"__global__[^;{]*\b" + name + r"\(", fn):
                return fn
    raise AssertionError(f"no kernel {name}")


def test_kernels_launched_as_programmatic_dependents_wait():
    """A kernel launched with ``launch_pdl`` may start while the one in front of it still runs: it
    has to wait for that kernel's results, and only then let the next one start."""
    names = set()
    for text in TEXTS.values():
        for fn in _functions(text):
            if "launch_pdl(" in fn:
                found = re.findall(r"\b\w+_kernel\b", fn)
                assert found, fn[:200]
                names.update(found)
    assert {"gelu_fwd_kernel", "gelu_bwd_kernel", "gemm_small_kernel", "qk_rope_bwd_kernel",
            "attn_fwd_pair_kernel", "rms_fwd_kernel"} <= names
    for name in sorted(names):
        body = _kernel_body(name)
        assert "pdl_wait();" in body, name
        assert 0 <= body.find("pdl_wait();") < body.find("pdl_trigger();"), name


def test_lanes_of_the_load_warp_of_dkv_agree_on_their_waits():
    """Every wait is bounded, and may run out in some lanes only: all 32 take part in the shuffles
    behind it, so they have to leave the loops together."""
    body = _kernel_body("attn_dkv_kernel")
    loads = body[body.index("if (warp == kDkvMath / 32) {"):
                 body.index("if (warp == kDkvMath / 32 + 1) {")]
    per_item, per_step = loads.split("i < steps && ok;")
    waits = re.findall(r"(.*)mbar_wait\(", per_item)
    assert len(waits) == 2 and all(w.endswith("__all_sync(0xffffffffu, ") for w in waits)
    # lanes that left the inner loop meet the others behind it
    behind = per_step[per_step.index("unsigned drawn"):]
    assert behind.index("ok = __all_sync(0xffffffffu, ok);") < behind.index("__shfl_sync")


def test_every_thread_of_the_small_gemm_waits_before_it_stores():
    """The loading and the issuing warp store results too, and a cluster barrier of the aligned form
    wants whole warps, which the loops in front of it do not leave together."""
    body = _kernel_body("gemm_small_kernel")
    joined = body[:body.index("sum and store")].rsplit("\n  }\n", 1)[1]    # behind the warps' roles
    assert "pdl_wait();" in joined
    text = next(t for t in TEXTS.values() if "void cluster_sync_()" in t)
    barrier = text[text.index("void cluster_sync_()"):]
    assert barrier.index("__syncwarp();") < barrier.index("barrier.cluster.arrive")


def _source(name):
    return next(text for p, text in TEXTS.items() if p.name == name)


def test_scales_are_written_behind_the_products_that_read_them():
    """A slot of scale words in tensor memory is written again once the products that read it are done: between the wait
    that says so and the store there is a fence."""
    for name, stores in (("gemm_block.cu", 3), ("gemm_block_2cta.cu", 2)):
        text = _source(name)
        found = [m.start() for m in re.finditer(r"tmem_st_32x32b_x\d\(tmem|tmem_st_32x32b_x\d\(dst|\"tcgen05\.st\.", text)]
        assert len(found) == stores, name
        for at in found:
            wait = max(text.rfind("mbar_wait(&sempty[", 0, at), text.rfind("mbar_wait(&empty[", 0, at))
            assert "tc_fence_after();" in text[wait:at], (name, text[at:at + 80])


def test_scales_of_the_second_cta_are_handed_over_across_the_cluster():
    """Tensor memory that a warp of the one CTA has written is read by products that a thread of the other issues: the
    arrival and the wait are at the scope of both, between the fences of tensor memory."""
    text = _source("gemm_block_2cta.cu")
    scales = text[text.index("tmem_st_32x32b_x8(dst"):text.index("if (w < last) {")]
    assert re.findall(r"tmem_st_wait|tc_fence_before|mbar_arrive\w*", scales) == ["tmem_st_wait", "tc_fence_before",
                                                                               "mbar_arrive_cluster"]
    (wait,) = re.finditer(r"mbar_wait\w*\(&sfull", text)
    assert wait.group() == "mbar_wait_cluster(&sfull"
    assert "tc_fence_after();" in text[wait.start():text.index("umma2_block(d_tmem")]
    pair = _source("pair.cuh")
    assert "mbarrier.arrive.relaxed.cluster.shared::cluster.b64" in pair
    assert "mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64" in pair
