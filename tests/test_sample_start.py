"""What orders the blocks of a row's cluster before they touch each other's shared
memory (kestrel_b200/csrc/sample.cu). CUDA asks that a block runs before a peer
writes to its shared memory; only the cluster's barrier tells. A model of the
blocks' first steps looks for an order in which a store comes before its target has
begun, and the kernel's text is held to the steps for which there is none."""
import os
import re

KERNEL = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kestrel_b200", "csrc", "sample.cu")


def early_store(steps, blocks):
    """Whether some order of the blocks' steps has a store to a block that has not
    begun. steps: "arrive", "wait" (for all to arrive), "store" (to every block)."""
    seen, todo = set(), [(0,) * blocks]  # a block's steps done; 0: it has not begun
    while todo:
        at = todo.pop()
        if at in seen:
            continue
        seen.add(at)
        for b in range(blocks):
            nxt = at[:b] + (at[b] + 1,) + at[b + 1:]
            if at[b] == 0:
                todo.append(nxt)
            elif at[b] <= len(steps):
                step = steps[at[b] - 1]
                if step == "store" and 0 in at:
                    return True
                if step == "wait" and any(x <= 1 + steps.index("arrive") for x in at):
                    continue
                todo.append(nxt)
    return False


def kernel_steps():
    """The first steps of the kernel's body, up to the first store to a peer."""
    with open(KERNEL) as f:
        body = f.read().split("sample_kernel(const SampleArgs a", 1)[1]
    out = []
    for m in re.finditer(r"cluster\.barrier_(arrive|wait)\(\)|in_block\(|x\.sync\(\)", body):
        out.append(m.group(1) or ("store" if m.group(0).startswith("in_block") else "sync"))
        if out[-1] == "store":
            return out
    return out


def test_a_barrier_is_needed():
    assert early_store(["store"], 2)
    assert early_store(["arrive", "store"], 3)
    assert not early_store(["arrive", "wait", "store"], 4)


def test_kernel_waits_for_its_peers_to_run():
    assert not early_store(kernel_steps(), 4)
