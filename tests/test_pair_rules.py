"""What a pair of blocks (tc05.cuh, namespace pair) owes each other, read from the sources: a kernel that broke it would
write into the shared memory of a block that has ended, and no test would see that on a GPU but now and then."""
import os
import re

from test_launch_rules import CSRC, _closing


def _source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def _branch(text, condition):
    """The statement's block behind if (condition), and the place where it ends."""
    at = text.index(f"if ({condition}) {{")
    at = text.index("{", at)
    end = _closing(text, at, "{}")
    return text[at:end + 1]


def test_arrivals_of_the_other_block_have_come_when_a_block_ends():
    """mma_commit arrives at barriers of both blocks.  bar_acc_full and the barriers of a stage that is loaded again are
    waited for on the way; those of the last stages are not, unless the loading warp of each block does so in the end."""
    text = _source("grouped.cu")
    body = text[text.index("grouped_kernel(const __grid_constant__"):text.index("join_kernel(")]
    committed = set(re.findall(r"mma_commit\(&(\w+)", body))
    assert committed == {"bar_empty", "bar_acc_full", "bar_drain"}  # the last one only when a wait ran out
    loader = body[body.index("warp == 0", body.index("auto next")) - 4:]
    loader = _branch(loader, "warp == 0")
    loop = loader.index("while (ok && next())")
    behind = loader[_closing(loader, loader.index("{", loop), "{}"):]
    assert re.search(r"for \([^)]*kStages[^)]*\)[^;]*mbar_wait\(&bar_empty\[", behind)
    epilogue = _branch(body, "warp >= kFirstEpilogue")
    assert "mbar_wait(&bar_acc_full[" in epilogue
