"""The no-hang contract of the prefill kernels, read from their source (a completion that never comes is
nothing a test can stage without hanging a kernel): a wait without a clock of its own ends only when another role raises the abort flag, so
behind each completion that such a wait depends on some role must wait with a clock."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash_attention_b200", "csrc")


def _role(name, banner):
    """The code of one role, from its banner to the next one, without comments."""
    text = open(os.path.join(CSRC, name)).read()
    parts = re.split(r"// =+ (.+?) =+\n", text)
    roles = {parts[i].strip(): parts[i + 1] for i in range(1, len(parts) - 1, 2)}
    return re.sub(r"//.*", "", roles[banner])


@pytest.mark.parametrize("name,banner", [("attn_ws64.cuh", "TMA loaders"), ("attn_ws.cuh", "PV issuer")])
def test_the_last_product_of_a_cta_is_awaited_with_a_clock(name, banner):
    """The last P V of a CTA's last tile: its reader waits by the flag alone, and no issuer has anything
    behind it to wait for.  One of the roles with a clock waits for it, after its tile loop and before its drain."""
    loop, drain = _role(name, banner).split("ti += 1;")
    tail = drain[:drain.index("kDrain")]
    assert re.search(r"\bmbar_wait(_relaxed<\w+>)?\(bars\.at\(Bars::kPvDone", tail), "no bounded wait behind the last product"
    assert "mbar_wait_flag" not in loop + drain


@pytest.mark.parametrize("name", ["attn_decode.cuh", "aux_kernels.cuh", "quantize.cuh"])
def test_the_other_kernels_wait_with_a_clock_only(name):
    assert "mbar_wait_flag" not in open(os.path.join(CSRC, name)).read()


def test_a_decode_warp_writes_only_its_own_hand_over_slot():
    """Slot (wg, wq) is read by warp wq of the other warpgroup, and only its own hand-over barrier orders that
    reader before the next write: a write by any other warp could come before the read."""
    text = re.sub(r"//.*", "", open(os.path.join(CSRC, "attn_decode.cuh")).read())
    writes = re.findall(r"if \(([^\n]*?)\) s_hand\[([^\n]+?)\] = ", text)
    assert len(writes) == text.count("s_hand[") - len(re.findall(r"= s_hand\[", text)) == 2
    k_max_rows, k_r = 32, 8
    for cond, index in writes:
        for wg in (0, 1):
            for wq in range(4):
                for lane in range(k_r):
                    env = {"wg": wg, "wq": wq, "lane": lane, "my_row": lane, "kR": k_r, "kMaxRows": k_max_rows}
                    if eval(cond.replace("&&", "and"), env):
                        assert eval(index, env) == (wg * 4 + wq) * k_max_rows + lane, (cond, index, wg, wq)


def test_accumulators_that_were_stored_are_awaited_before_they_are_read_again():
    """Many rows over the 8-bit cache: a row's reference may move in both halves of a step, and tensor-memory stores and
    loads of one thread are ordered by tcgen05.wait alone.  Behind each loop that stores O stands a wait for its stores."""
    text = re.sub(r"//.*", "", open(os.path.join(CSRC, "fp8_prefill.cuh")).read())
    stores = [m.end() for m in re.finditer(r"tmem_st\d+\(tm_o\b[^;]*;", text)]
    assert stores
    for at in stores:
        rest = text[at:]
        wait = rest.index("tc_wait_st()")
        assert "tmem_ld" not in rest[:wait] and re.fullmatch(r"\s*}\s*", rest[:wait])


def test_products_wait_for_what_they_overwrite():
    """Many rows over the 8-bit cache: tensor memory that one product reads and another overwrites.  Products of different accumulators may run in
    any order, so the scores of step i + 1 go to the half of the columns that W V of step i does not read, and each product that writes there waits for
    what was there: the weights of step i - 1 (W V done), the upper scores (taken by the softmax) for the lower ones."""
    loop = _role("fp8_prefill.cuh", "products")
    loop = loop[loop.index("uint32_t buf = 0"):]
    assert "half = (i + 1) & 1;" in loop and re.search(r"from = [^;]*\+ 64 \* \(i & 1\);", loop)
    assert re.search(r"gone = bar\(i == 0 \? L::kUFree : L::kPvDone\)", loop)
    waits = r"mbar_wait\(%s, %s, wc, \w+\)"
    first, second = [m.start() for m in re.finditer(r"score\(", loop)]
    assert "true, half" in loop[first:first + 40] and "false, half" in loop[second:second + 40]
    assert re.search(waits % ("gone", "phase"), loop[:first]) and re.search(waits % (r"gone \+ 8 \* two", "phase"), loop[:first])
    assert re.search(waits % (r"bar\(L::kUFree \+ t\)", "half") + r";\s*if \(!ok\) break;\s*tc_fence_after_sync\(\);\s*$", loop[:second])


@pytest.mark.parametrize("banner", ["Q . K^T", "V^T . W^T"])
def test_products_over_the_8_bit_cache_are_awaited_whoever_gave_up(banner):
    """An issuer may have nothing left to wait for when another role's wait runs out: its last products are on their way then, and
    the CTA's memory must not be released before them."""
    role = _role("fp8_decode.cuh", banner)
    drain = role.rindex("tc_commit(bar(F::kDrain")
    assert "if (!ok) {" not in role and re.search(r"const uint64_t begun = globaltimer_ns\(\);\s*$", role[:drain])


def test_copies_of_the_8_bit_cache_are_awaited_whoever_gave_up():
    for name, calls in (("fp8_decode.cuh", 1), ("fp8_prefill.cuh", 2)):
        text = re.sub(r"//.*", "", open(os.path.join(CSRC, name)).read())
        assert len(re.findall(r"^ *feed\.drain\(\);$", text, re.M)) == text.count("feed.drain()") == calls
