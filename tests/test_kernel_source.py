"""Orderings and ways out of the kernels that no run can show reliably, read from their source."""

import pathlib
import re

CSRC = pathlib.Path(__file__).resolve().parent.parent / "fp8-replayssm-gdn-kernel_b200" / "csrc"


def source(name):
    """A source file without comments."""
    text = (CSRC / name).read_text()
    return re.sub(r"/\*.*?\*/", "", re.sub(r"//[^\n]*", "", text), flags=re.S)


def block(text, head):
    """What follows ``head``, to the brace that closes the first one opened behind it."""
    assert text.count(head) == 1, (head, text.count(head))
    at = text.index("{", text.index(head) + len(head))
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i + 1]
    raise AssertionError(head)


def body(text, function):
    """Body of the kernel or function of that name (its definition ends in an opening brace)."""
    heads = re.findall(r"[^;}]*\b%s\([^;{]*\)\s*(?:const\s*)?(?=\{)" % function, text)
    assert len(heads) == 1, (function, heads)
    return block(text, heads[0].strip())


def test_output_staged_over_a_tile_is_fenced_before_the_tile_is_given_back():
    """Ordinary stores into memory that TMA writes next: a proxy fence between them and the arrival that frees it."""
    finish = block(body(source("gdnr_prefill.cu"), "prefill_scan_tc_kernel"), "auto finish = ")
    stored = finish.rindex("reinterpret_cast<uint16_t*>(v + swz")
    freed = finish.index("mbar_arrive(&sm.empty")
    assert "fence.proxy.async.shared::cta" in finish[stored:freed]


def test_consumers_of_attention_leave_together():
    """A warp whose bounded wait gave up must not leave while others go on to a barrier that counts it: between a wait and the next
    barrier there is no way out, and that barrier tells all of them."""
    consumers = block(body(source("gdnr_attn.cu"), "attn_stream_kernel").split("const int wm = warp / WN")[1], "for (int64_t at = share.begin")
    tiles = block(consumers, "for (int t = t0; t < t1; ++t, ++k)")
    assert re.search(r"ok = wait\(&full\[st\][^;]*;\s*if \(!ok\) break;", tiles)
    assert "bar_sync" not in tiles
    returns = re.findall(r"if \(([^;{}]*)\)\s*return;", consumers)
    assert len(returns) == consumers.count("return") and all(r.startswith("bar_or(1, C::CONSUMERS, ") for r in returns), returns
    after = consumers[consumers.index(tiles) + len(tiles):]
    assert re.match(r"[^;]*\bfor [^{]*\{[^}]*\}\s*if \(bar_or\(1, C::CONSUMERS, !ok\)\) return;", after), after[:300]


def test_copies_in_flight_land_whoever_gave_up():
    """A warp that requests tiles waits for the last of them also where its own waits were all met: no condition before it."""
    attn, tc, prefill = (source(f) for f in ("gdnr_attn.cu", "gdnr_attn_tc.cu", "gdnr_prefill.cu"))
    for text, kernel, drains in ((attn, "attn_stream_kernel", ["drain(full, STAGES, k);"]),
                                 (tc, "attn_tc_kernel", ["drain(&bars.q_full[q], 1, nq[q]);", "drain(bars.kv_full, C::RING, slot);"]),
                                 (prefill, "prefill_scan_kernel", ["drain(sm.full, CS_STAGES, c);"]),
                                 (prefill, "prefill_scan_tc_kernel", ["drain(sm.full, CS_STAGES, c);"])):
        for drain in drains:
            before = body(text, kernel).split(drain)
            assert len(before) == 2, (kernel, drain)
            assert not re.search(r"if \([^)]*\)\s*$", before[0]), (kernel, before[0][-80:])
    derive = body(prefill, "prefill_derive_kernel")
    assert "drain(&sm.bar, 1, 1);" in block(derive, "if (__syncthreads_or(!ok)) ")


def test_a_wait_looks_once_more_before_it_reports_a_timeout():
    """The clock may have run out because the waiting thread itself was held up, with the barrier complete meanwhile."""
    for name, wait in (("gdnr_tile.cuh", "slow"), ("gdnr_device.cuh", "mbar_wait_bounded")):
        text = body(source(name), wait)
        behind = text[text.index(block(text, "for (")):]
        assert "if (mbar_try_wait(a, parity)) return true;" in behind[len(block(text, "for (")):behind.index("atomicOr")], name


def test_every_share_leaves_a_record_for_the_join():
    """The join reads a record of each CTA from a workspace that holds anything: no way out before it is written."""
    for name, kernel in (("gdnr_attn.cu", "attn_kernel"), ("gdnr_attn.cu", "attn_stream_kernel"), ("gdnr_attn_tc.cu", "attn_tc_kernel")):
        text = body(source(name), kernel)
        before = re.split(r"write_meta<T>|WarpWait wait\{", text)[0].split("return;")
        for way_out in before[:-1]:
            assert "meta[0] = -1" in way_out, (kernel, way_out[-200:])
    tc = body(source("gdnr_attn_tc.cu"), "attn_tc_kernel")
    assert re.search(r"write_meta<T>[^}]*\}\s*else if \(tid == 0\) \{\s*meta\[0\] = -1;", tc)


def test_a_chunk_without_images_stops_the_scan():
    """Where the first kernel's wait gave up the workspace holds anything: it says so, and neither scan stores a state made of it."""
    text = source("gdnr_prefill.cu")
    assert re.search(r"->made = 0;", block(body(text, "prefill_derive_kernel"), "if (__syncthreads_or(!ok)) "))
    assert "img.made = 1;" in body(text, "prefill_derive_kernel")
    for kernel, agreed in (("prefill_scan_kernel", "bar_or("), ("prefill_scan_tc_kernel", "announce(&sm.s_ready)")):
        scan = body(text, kernel)
        looked = scan.index("im.made")
        assert looked < scan.index(agreed), kernel
        assert re.search(r"if \(!ok\) (break|return);", scan[looked:scan.index(agreed) + 200]), kernel
    assert re.search(r"if \(!ok\) return;\s*#pragma unroll", body(text, "prefill_scan_kernel"))
    assert re.search(r"if \(ok\) \{\s*tc_fence_after", body(text, "prefill_scan_tc_kernel"))


def test_null_slot_rows_are_counted_in_tokens():
    """A sequence's values pass 2^31 before its tokens do (up to 2^30 of them are taken): the loop counts tokens."""
    text = source("gdnr_prefill.cu")
    for kernel in ("prefill_scan_kernel", "prefill_scan_tc_kernel"):
        zeros = block(body(text, kernel), "if (r.slot < 0) ")
        assert re.findall(r"for \([^)]*\)", zeros) == [re.search(r"for \(int t = r\.begin \+ warp; t < r\.end; t \+= [^)]*\)", zeros)[0]], kernel


def test_error_word_address_is_not_kept():
    """It belongs to the device's context: an address kept over a reset would be written to by the next call's kernel."""
    lookup = body(source("gdnr_api.cu"), "default_error_word")
    assert "cudaGetSymbolAddress" in lookup and "static" not in lookup.replace("static_cast", "")
