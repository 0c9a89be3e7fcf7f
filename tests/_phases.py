"""Barriers that are waited for by parity, as a graph of what comes before what.

Events are tuples: ("done", barrier, phase) completes a phase, ("seen", barrier, phase, who) is a wait for
it that is over, ("set", barrier, phase) announces a copy that will complete it.  Edges are program order in
each role, and from what completes a phase to whoever waits for it; what follows from them holds
whatever anything takes.  A barrier is named by what it counts; the phase after n on the same barrier is
n + step(barrier)."""


class Graph:
    def __init__(self, step):
        self.before = {}
        self.role = {}  # a wait -> what its role did before it
        self.step = step

    def event(self, e, *after):
        self.before.setdefault(e, set()).update(a for a in after if a is not None)
        return e

    def wait(self, bar, phase, who, last):
        e = ("seen", bar, phase, who)
        self.role.setdefault(e, last)
        return self.event(e, last, ("done", bar, phase))

    def ancestors(self):
        """Every event's ancestors, as a set."""
        memo, state = {}, {}
        for root in list(self.before):
            stack = [root]
            while stack:
                e = stack[-1]
                if e in memo:
                    stack.pop()
                    continue
                missing = [a for a in self.before.get(e, ()) if a not in memo]
                if missing and state.get(e) != "open":
                    state[e] = "open"
                    stack.extend(missing)
                    continue
                assert not missing, f"{e} waits for itself"
                memo[e] = set().union(*({a} | memo[a] for a in self.before.get(e, ())))
                stack.pop()
        return memo

    def faults(self, anc):
        """Waits and announcements that only timing keeps right."""
        found = []
        for e in anc:
            if e[0] not in ("set", "seen"):
                continue
            ahead = ("done", e[1], e[2] - self.step(e[1]))
            if e[0] == "set" and ahead in anc and ahead not in anc[e]:
                found.append(f"{e[1]} {e[2]} announced while the copy before it may be on its way")
            if e[0] == "seen":
                last = self.role[e]
                if ahead in anc and (last is None or ahead not in anc[last] | {last}):
                    found.append(f"{e[1]} {e[2]} may seem over to {e[3]} while the phase before it is not")
                following = ("done", e[1], e[2] + self.step(e[1]))
                if following in anc and e not in anc[following]:
                    found.append(f"{e[1]} {e[2]} may be over and gone before {e[3]} has seen it")
        return found
