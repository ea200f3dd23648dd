"""Drafts for greedy decoding without a second model: continuations that
followed earlier occurrences of the last tokens, as a tree, and the walk that
accepts what the model agrees with.  Host code, one sequence at a time.
"""
from __future__ import annotations

__all__ = ["TextIndex", "draft_tree", "accept"]


class TextIndex:
    """A text that grows, and where each of its n-grams (n <= ``max_ngram``)
    begins, so that a step does not search the whole text for its last tokens."""

    def __init__(self, tokens: list[int], max_ngram: int = 3):
        self.tokens: list[int] = []
        self.max_ngram = max_ngram
        self._starts: list[dict[tuple, list[int]]] = [{} for _ in range(max_ngram)]
        self.extend(tokens)

    def __len__(self) -> int:
        return len(self.tokens)

    def extend(self, tokens: list[int]) -> None:
        old = len(self.tokens)
        self.tokens += tokens
        for n, starts in enumerate(self._starts, 1):
            for start in range(max(0, old - n + 1), len(self.tokens) - n + 1):
                starts.setdefault(tuple(self.tokens[start:start + n]), []).append(start)

    def earlier(self, n: int):
        """Where the last ``n`` tokens occurred before, the latest first."""
        starts = self._starts[n - 1][tuple(self.tokens[-n:])]
        return (starts[i] for i in range(len(starts) - 2, -1, -1))


def draft_tree(text: TextIndex | list[int], size: int, branches: int = 4) -> tuple[list[int], list[int]]:
    """A tree of at most ``size`` nodes that continues ``text``: (token of each
    node, parent of each node).  Node 0 is the last token (parent -1); the rest
    are the tokens behind up to ``branches`` earlier occurrences of the last
    ``text.max_ngram`` (then fewer) tokens, the latest occurrences first, merged where
    they begin alike.  Parents come before their children."""
    if not isinstance(text, TextIndex):
        text = TextIndex(text)
    tokens = text.tokens
    nodes, parents = [tokens[-1]], [-1]
    children: dict[tuple[int, int], int] = {}  # (parent, token) -> node
    found = 0
    for n in range(min(text.max_ngram, len(tokens) - 1), 0, -1):
        for start in text.earlier(n):
            if len(nodes) >= size or found >= branches:
                return nodes, parents
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
