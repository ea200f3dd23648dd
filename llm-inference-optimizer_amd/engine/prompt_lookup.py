"""Drafts for greedy decoding without a second model: continuations that
followed earlier occurrences of the last tokens, as a tree, and the walk that
accepts what the model agrees with.  Host code, one sequence at a time.
"""
from __future__ import annotations

__all__ = ["draft_tree", "accept"]


def draft_tree(tokens: list[int], size: int, max_ngram: int = 3, branches: int = 4) -> tuple[list[int], list[int]]:
    """A tree of at most ``size`` nodes that continues ``tokens``: (token of each
    node, parent of each node).  Node 0 is the last token (parent -1); the rest
    are the tokens behind up to ``branches`` earlier occurrences of the last
    ``max_ngram`` (then fewer) tokens, the latest occurrences first, merged where
    they begin alike.  Parents come before their children."""
    nodes, parents = [tokens[-1]], [-1]
    children: dict[tuple[int, int], int] = {}  # (parent, token) -> node
    found = 0
    for n in range(min(max_ngram, len(tokens) - 1), 0, -1):
        suffix = tokens[-n:]
        for start in range(len(tokens) - n - 1, -1, -1):
            if len(nodes) >= size or found >= branches:
                return nodes, parents
            if tokens[start:start + n] != suffix:
                continue
            found += 1
            at = 0
            # half of the free nodes for each continuation but the last: room for others
            room = max(1, (size - len(nodes) + 1) // 2) if found < branches else size - len(nodes)
            for token in tokens[start + n:start + n + size]:
                key = (at, token)
                if key not in children:
                    if room == 0 or len(nodes) >= size:
                        break
                    room -= 1
                    children[key] = len(nodes)
                    nodes.append(token)
                    parents.append(at)
                at = children[key]
        if found:
            break
    return nodes, parents


def accept(nodes: list[int], parents: list[int], picks: list[int]) -> list[int]:
    """The path of nodes, from node 0 on, whose tokens are the model's own picks
    (``picks[i]``: its next token after node i); the pick after the last is new."""
    path = [0]
    while True:
        nxt = next((i for i in range(path[-1] + 1, len(nodes)) if parents[i] == path[-1] and nodes[i] == picks[path[-1]]),
                   None)
        if nxt is None:
            return path
        path.append(nxt)
