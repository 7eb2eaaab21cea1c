"""What the attention kernels with tiles on the tensor core do when a wait runs out, read from the sources (no run may make one run out): nothing is copied or multiplied behind
it, and what was begun ends before the CTA gives its tensor memory and shared memory back."""
import os
import re

from test_launch_order_cpu import CSRC, functions

TAKES = re.compile(r"mbar_expect_tx\(|bulk_g2s\(|tc_mma_f16_ts<|atc_mma_ss<")


def body(name):
    return functions()[name][2]


def looked_at(text, doers):
    """Every one of doers behind a wait has a look at that wait's outcome in front of it; how many there are."""
    n = 0
    for m in re.finditer(doers, text):
        before = text[:m.start()]
        waits = list(re.finditer(r"\bwait\(", before))
        if waits:
            n += 1
            assert re.search(r"if \(!ok\) (?:return|break);", before[waits[-1].start():]), text[waits[-1].start():m.end() + 40]
    return n


def test_uses_in_turn():
    """The number of uses that a barrier had, by which the last one's parity is found."""
    rule = re.search(r"int in_turn\(int n, int m, int c\) \{ return (.*?); \}", open(os.path.join(CSRC, "common.cuh")).read())[1].replace("/", "//")
    for m in (1, 2, 4):
        for n in range(40):
            used = [0] * m
            for i in range(n):
                used[i % m] += 1
            assert used == [eval(rule, {"n": n, "m": m, "c": c}) for c in range(m)]


def test_shared_pages():
    text = body("pst_drivers")
    assert looked_at(text, TAKES) >= 8
    # pages that are multiplied: none behind a wait that ran out; parts that are copied: none, and as many counted as were begun
    assert len(re.findall(r"i < \w+ && ok; \+\+i, \+\+it", text)) == 2 and len(re.findall(r"\+\+i, \+\+begun\)", text)) == 2
    # each warp's way out: products that were issued, copies that were begun
    assert re.search(r"products_end\(done\);\s*return;", text) and "products_end(done + 1)" in text
    assert "copies_end(begun, vfull, 2, gfull)" in text and "copies_end(begun, kfull, 4, ffull)" in text
    assert not re.search(r"\*failed\) return", text)
    for end in ("copies_end", "products_end"):
        assert "psh_wait" in re.search(end + r" = \[&\](.*?)\n    \};", text, re.S)[1]
    # the barriers that the products end on are begun, and no two of the barriers are one
    kernel = body("pages_shared_tc_kernel")
    assert "b < PST_BARS" in kernel and "qk + PST_BARS" in kernel
    at = [(int(x), n) for n, x in re.findall(r"\*(\w+) = qk \+ (\d+)", text)]
    size = {"vfull": 2, "kfull": 4, "kfree": 4, "ffull": 2, "vfree": 2, "gfull": 2, "done": 2}
    used = [b for first, n in at for b in range(first, first + size.get(n, 1))]
    bars = int(re.search(r"PST_BARS = (\d+)", open(os.path.join(CSRC, "pages_shared_tc.cuh")).read())[1])
    assert sorted([0, *used]) == list(range(bars))


def test_pages_of_one_sequence():
    text = body("pages_tc_kernel")
    driver = text[text.index("if (driver) {"):]
    driver = driver[:driver.index("return;\n    }\n    {")]
    assert looked_at(driver, r"\b(?:load_[kv]|issue_(?:qk|pv))\(") == 4
    assert re.search(r"tc_commit\(done\);\s*__syncwarp\(\);\s*mbar_wait_try\(done, 0\);", driver)
    # the last copy of each barrier, by its parity: copy i is use i >> 1 of barrier i & 1
    ends = re.findall(r"if \(i > (\d)\) mbar_wait_try\(full \+ (\(.*?\)), \(uint32_t\)\((.*?)\)\);", driver)
    for i in range(12):
        last = {j & 1: (j >> 1) & 1 for j in range(i)}
        assert {eval(bar, {"i": i}): eval(parity, {"i": i}) for least, bar, parity in ends if i > int(least)} == last
    assert "*done = qk + 8;" in text and "b < 9" in text and "done + 1" in text


def test_a_prompt_by_itself():
    text = body("attn_tc_kernel")
    loop = text[text.index("for (int i = 0; i < ntiles; ++i)"):]
    end = loop.index("if (!__syncthreads_and(ok ? 1 : 0)) {")
    # products and copies: by a thread none of whose waits has run out, or behind a barrier that says so of all
    assert re.search(r"[^\n]*load_v\(i \+ 1\)", loop[:end])[0].count("&& ok)") == 1
    assert text.count("if (elect_one() && ok)") == 5 and text.count("elect_one()") == 6
    assert loop.index("if (!__syncthreads_and(ok ? 1 : 0)) break;") < loop.index("load_k(i + 1)")
    way_out = loop[end:loop.index("red[cg * ATC_M + row] = l_run;")]
    assert re.search(r"tc_commit\(done\);\s*__syncwarp\(\);\s*mbar_wait_try\(done, 0\);", way_out) and way_out.rstrip().endswith("__syncthreads();\n    }")
    assert "mbar_init(done, 2);" in text
    assert re.findall(r"mbar_wait_try\(full, (\d)\)", way_out) == ["0", "1"] and "warp == 4 ? kfull : vfull" in way_out


def test_pages_in_slots():
    """A barrier that counts a copy is arrived at once a phase, and what a fragment is said to be is not written over while it may be read: neither behind a wait that ran out."""
    source = open(os.path.join(CSRC, "pages_shared.cuh")).read()
    load = source[source.index("__device__ __forceinline__ void load(const PshFragment &F)"):]
    load = load[:load.index("void end()")]
    wait = load.index("wait(&empties[j]")
    look = load.index("if (!wait.ok) break;", wait)
    assert all(look < load.index(x) for x in ("mbar_expect_tx(&fulls[j]", "mbar_arrive(&fulls[j])", "bulk_g2s(")) and "++p, ++n)" in load[:wait]
    say = body("psh_plan_warp")
    say = say[say.index("auto say = "):]
    assert say.index("wait(&S.dempty") < say.index("if (!wait.ok) return;") < say.index("S.desc[said % PSH_DESCS] = F;")
