"""Drafted tokens: what a request's own tokens say may come next.

Text repeats itself (quotations, code, lists, names): where the last few tokens stood before, what followed them then is a
guess at what follows now.  `PromptLookup` keeps, per request, the places of every run of 1 to `longest` tokens and proposes
the continuations behind the latest places of the longest run that has any, as a tree whose root is the last token.  A guess
costs rows of the step that checks it (`Engine.step_drafts`): what the model does not say itself is dropped, so the
tokens of a request are those that it has without drafts, up to the rounding of a step with more rows (in float32 the last bits).

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
        # by a run's length: the run -> the indexes behind its latest places, oldest first (one place is a number by itself: most
        # runs have no more, and a prompt's tokens are many: 32,000 take 25 ms so, 120 with a list for each)
        self._places: list[dict] = [{} for _ in range(longest)]

    def extend(self, tokens) -> None:
        """The request goes on with these tokens."""
        known, first = self.tokens, len(self.tokens)
        known.extend(int(t) for t in tokens)
        keep = -(self.branches + 1)                      # (the last one is the end itself, behind which nothing is known)
        for n, places in enumerate(self._places, 1):
            runs = known[max(first - n + 1, 0) :]
            for end, run in enumerate(runs if n == 1 else zip(*(runs[i:] for i in range(n))), max(first + 1, n)):
                before = places.get(run)
                if before is None:
                    places[run] = end
                elif type(before) is int:
                    places[run] = (before, end)[keep:]
                else:
                    places[run] = (*before, end)[keep:]

    def _behind(self, n: int) -> list[int]:
        """The indexes behind the latest places of the last n tokens, oldest first, their own place aside."""
        end = len(self.tokens)
        places = self._places[n - 1].get(self.tokens[-1] if n == 1 else tuple(self.tokens[end - n :]), ())
        return [p for p in ((places,) if type(places) is int else places) if p < end]

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
            places = self._behind(n)
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
