"""Kernels that may start before the one ahead of them in their stream has ended, read as text: each waits for that kernel before it lets the next one in, and before it
touches memory that another kernel may write."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'hopper_megamoe_basedondeepgemm_b200', 'csrc')


def _block(text, at):
    """Where the block that opens at `at` ends."""
    depth = 0
    for end in range(at, len(text)):
        depth += {'{': 1, '}': -1}.get(text[end], 0)
        if depth == 0:
            return end + 1


def _kernels():
    """(name, body without comments) of every kernel in the sources."""
    found = []
    for path in sorted(glob.glob(os.path.join(CSRC, '*.cu*'))):
        with open(path) as f:
            text = re.sub(r'//[^\n]*|/\*.*?\*/', '', f.read(), flags=re.S)
        for m in re.finditer(r'__global__\s+void\b', text):
            name = re.compile(r'(\w+)\s*\(\s*(?:const\s+)?(?:__grid_constant__\s+)?[\w:]*Params').search(text, m.end())
            if name is None or name.start() - m.end() > 300:
                continue
            at = text.index('{', name.end())
            found.append((name.group(1), text[at:_block(text, at)]))
    return found


KERNELS = [(n, b) for n, b in _kernels() if 'grid_launch_dependents' in b]


def test_there_are_kernels_that_start_early():
    names = {n for n, _ in KERNELS}
    assert {'balance_kernel', 'balance_zero_kernel', 'balance_small_kernel', 'route_kernel', 'router_backward_kernel', 'block_norm_kernel', 'block_norm_backward_kernel',
            'block_norm_sums_kernel'} <= names, names


@pytest.mark.parametrize('name, body', KERNELS, ids=[n for n, _ in KERNELS])
def test_a_kernel_waits_before_it_lets_the_next_one_in(name, body):
    while (m := re.search(r'= \[&\]\([^)]*\) \{', body)) is not None:      # (a lambda runs where it is called)
        body = body[:m.start()] + body[_block(body, m.end() - 1):]
    wait, lets = body.find('grid_dependency_wait()'), body.find('grid_launch_dependents()')
    assert 0 <= wait < lets
    assert not re.search(r'\b(?:fetch\w*|rt_fetch|rt_balance_\w+|bn_fetch|bn_sum\w*)\s*(?:<[^;(]*>)?\s*\(', body[:wait])
    assert body.count('grid_dependency_wait()') == 1 and body.count('grid_launch_dependents()') == 1
