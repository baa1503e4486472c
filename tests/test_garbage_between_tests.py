"""What a test leaves in reference cycles (an engine whose group holds a closure over
itself, with its device memory) is gone when the next test begins, and not freed
somewhere inside it: tests of the allocator's counts rely on that."""

from __future__ import annotations

import weakref


class Node:
    pass


_left = []


def test_one_leaves_a_cycle():
    node = Node()
    node.itself = node
    _left.append(weakref.ref(node))


def test_the_next_does_not_see_it():
    assert all(ref() is None for ref in _left)
