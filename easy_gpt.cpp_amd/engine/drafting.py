"""Drafted tokens: what a request's own tokens say may come next.

Text repeats itself (quotations, code, lists, names): where the last few tokens stood before, what followed them then is a
guess at what follows now.  `PromptLookup` keeps, per request, the places of every run of 1 to `longest` tokens and proposes
the continuations behind the latest places of the longest run that has any, as a tree whose root is the last token.  A guess
costs nothing but rows of the step that checks it (`Engine.step_drafts`): what the model does not say itself is dropped, so the
tokens of a request are those that it has without drafts.

The reference decodes one token per request and step (/root/reference/src/continuous_batch_server.cpp:160-212).
"""
from __future__ import annotations

from .. import kernels


class PromptLookup:
    """The places of a request's runs of tokens, brought up to date by `extend`."""

    def __init__(self, longest: int = 3, branches: int = 3):
        if longest < 1 or branches < 1:
            raise ValueError("longest and branches must be greater than 0")
        self.longest, self.branches = longest, branches
        self.tokens: list[int] = []
        self._places: dict[tuple, list[int]] = {}        # a run -> the indexes behind its latest places, oldest first

    def extend(self, tokens) -> None:
        """The request goes on with these tokens."""
        for t in tokens:
            self.tokens.append(int(t))
            end = len(self.tokens)
            for n in range(1, min(self.longest, end) + 1):
                places = self._places.setdefault(tuple(self.tokens[end - n :]), [])
                places.append(end)
                if len(places) > self.branches + 1:      # (the last one is the end itself, behind which nothing is known)
                    del places[0]

    def propose(self, max_nodes: int, max_depth: int) -> tuple[list[int], list[int]]:
        """(tokens, parents) of a tree of at most max_nodes nodes, none deeper than max_depth: node 0 is the request's last
        token, with parent -1, and a child lies behind its parent."""
        end = len(self.tokens)
        if end == 0:
            raise ValueError("a request without tokens has nothing that could go on")
        max_nodes = min(max_nodes, kernels.KernelBackend.max_tree_nodes)
        tokens, parents = [self.tokens[-1]], [-1]
        children: dict[tuple[int, int], int] = {}
        for n in range(min(self.longest, end), 0, -1):
            places = [p for p in self._places.get(tuple(self.tokens[end - n :]), ()) if p < end]
            for p in reversed(places):                   # the latest first
                node = 0
                for t in self.tokens[p : p + max_depth]:
                    child = children.get((node, t))
                    if child is None:
                        if len(tokens) >= max_nodes:
                            break
                        child = children[node, t] = len(tokens)
                        tokens.append(t)
                        parents.append(node)
                    node = child
            if places:
                break
        return tokens, parents
