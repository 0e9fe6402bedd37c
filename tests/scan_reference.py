"""The gated recurrence row after row in float64, with a bound on what a kernel that composes its rows in fp32 may be off.

A gate's decay a, and 1 - a, are off by some six units of 2^-24 of themselves, a product or sum by one: a step adds STEP units of
the magnitudes in it, and an error decays as the state does, so that it follows the same recurrence as the magnitudes.  What is
composed of several rows goes through up to 8 + 8 + 4 + 16 further products, and one more for every tile of a run.

The exponential's results below 2^-126, the least normal number, are zero: a decay may be off by that much, and a gate's gradient,
which is a product with its decay, by that times the other factors (of a gate of -87.54, whose decay is 9.6e-39: -6.5e-38)."""
import numpy as np

UNIT = 2.0 ** -24
STEP, JOINS, NORMAL = 10, 64, 2.0 ** -126


def decays(g, kind):
    if kind == "exp":
        return np.exp(g), np.ones_like(g)
    return 1.0 / (1.0 + np.exp(-g)), 1.0 / (1.0 + np.exp(g))


def scan(x, g, starts, initial, kind, reverse, dh=None, df=None):
    """{name: (value, bound)} of out, final and, with dh, features_grad, gates_grad, initial_grad"""
    rows, channels = x.shape
    samples = len(starts) - 1
    a, u = decays(g, kind)
    h, he, prev, preve = (np.zeros_like(x) for _ in range(4))
    l, le = np.zeros_like(x), np.zeros_like(x)
    final, finale, di, die = (np.zeros((samples, channels)) for _ in range(4))
    for s in range(samples):
        way = list(range(starts[s], starts[s + 1]))
        if reverse:
            way.reverse()
        joins = JOINS + len(way) / 256 / 16
        at = initial[s].copy() if initial is not None else np.zeros(channels)
        size, room = np.abs(at), np.zeros(channels)
        for t in way:
            prev[t], preve[t] = at, (room + joins * size) * UNIT
            # (errors in units: those so far decay, and the step's own come on top)
            room = a[t] * (room + STEP * size) + STEP * np.abs(u[t] * x[t])
            size = a[t] * size + np.abs(u[t] * x[t])
            at = a[t] * at + u[t] * x[t]
            h[t], he[t] = at, (room + joins * size) * UNIT
        final[s], finale[s] = at, (room + joins * size) * UNIT
        if dh is None:
            continue
        at = df[s].copy() if df is not None else np.zeros(channels)
        size, room = np.abs(at), np.zeros(channels)
        for t in reversed(way):
            at, size, room = dh[t] + at, np.abs(dh[t]) + size, room + np.abs(dh[t]) + size
            l[t], le[t] = at, (room + joins * size) * UNIT
            at, size, room = a[t] * at, a[t] * size, a[t] * (room + STEP * size)
        di[s], die[s] = at, (room + joins * size) * UNIT
    found = {"out": (h, he), "final": (final, finale)}
    if dh is not None:
        found["features_grad"] = (u * l, u * (le + STEP * UNIT * np.abs(l)))
        inner, innere = (prev - x, preve + UNIT * (np.abs(prev) + np.abs(x))) if kind == "sigmoid" else (prev, preve)
        slope = a * u
        found["gates_grad"] = (l * inner * slope,
                               slope * (le * np.abs(inner) + np.abs(l) * (innere + 2 * STEP * UNIT * np.abs(inner))) +
                               NORMAL * np.abs(l * inner))
        found["initial_grad"] = (di, die)
    return found
