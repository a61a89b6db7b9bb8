"""What kernels do when a bounded wait runs out, read off their source: nothing may make a wait run out on a GPU that others share."""
import re
from pathlib import Path

KERNELS = Path(__file__).resolve().parent.parent / "tips_b200" / "csrc" / "kernels"


def test_attention_hands_nothing_on_after_a_failed_wait():
    """In the forward kernel a warp whose wait failed goes on to its next piece; probabilities or outputs that it signalled then would
    reach memory although the launch is reported as failed."""
    source = (KERNELS / "attention.cu").read_text()
    body = source[source.index("AttnFwdKernel("):source.index("// ---------------------------------------------------------------- backward")]
    softmax = body[body.index("Waiter wait(4);"):]
    arrivals = re.findall(r"if \(([^;]*)\) BarArrive\(([^;]*)\);", softmax)
    assert {bar for _, bar in arrivals} == {"p_full", "base + Cfg::kOStaged + i * 8"}
    assert all("wait.ok" in condition for condition, _ in arrivals)
    assert softmax.count("BarArrive(") == len(arrivals)
    stores = re.findall(r"if \(([^;]*)\)\s*(?:StoreCols|StoreRest|p\.lse\[)", softmax)
    assert len(stores) == 3 and all("wait.ok" in condition for condition in stores)


def test_epilogue_warps_decide_on_a_failed_wait_as_a_whole():
    """What follows the wait for an accumulator are instructions of a whole warp (loads from TMEM, votes, barriers): lanes that went on
    alone would wait for those that did not."""
    for name in ("gemm_tcgen05.cu", "conv_tcgen05.cu"):
        waits = re.findall(r"(\w+)\(&?tmem_full\b[^;{]*\)", (KERNELS / name).read_text())
        waits = [w for w in waits if w.startswith("Mbar") and "Wait" in w]
        assert len(waits) == 4 and set(waits) == {"MbarWaitWarp"}, name
