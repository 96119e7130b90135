"""What stands around a model's layers in a step, in 64 bits on the host: adjusted logits, truncated draws, block tables and the
index arrays of a step.  One loop per definition."""
import math

import numpy as np


def adjust(logits, row_seat=None, marks=None, counts=None, repetition=None, presence=None, frequency=None, bias=None, allowed=None,
           allowed_row=None):
    """(adjusted logits in 64 bits, a bound on what 32-bit arithmetic may be off by): every operation is off by at most 2^-24 of the
    largest number it can meet, and there are at most three and one per bias."""
    x = np.asarray(logits, dtype=np.float64).copy()
    rows, vocab = x.shape
    size, steps = np.abs(x), np.zeros_like(x)
    for r in range(rows):
        seat = -1 if row_seat is None else int(row_seat[r])
        lost = row_seat is not None and (seat < -1 or seat >= marks.shape[0])
        if seat >= 0 and not lost:
            for t in np.nonzero(marks[seat])[0]:
                if repetition is not None:
                    rep = float(repetition[r])
                    x[r, t] = x[r, t] / rep if x[r, t] > 0 else x[r, t] * rep
                    size[r, t] = abs(x[r, t])
                    steps[r, t] += 1
                c = 0 if counts is None else int(counts[seat, t])
                if c > 0:
                    f = 0.0 if frequency is None else float(frequency[r])
                    p = 0.0 if presence is None else float(presence[r])
                    x[r, t] -= f * c + p
                    size[r, t] += abs(f) * c + abs(p)
                    steps[r, t] += 2
        if bias is not None:
            start, token, value = bias
            for i in range(max(0, int(start[r])), min(len(token), int(start[r + 1]))):
                t = int(token[i])
                if 0 <= t < vocab:
                    x[r, t] += float(value[i])
                    size[r, t] += abs(float(value[i]))
                    steps[r, t] += 1
        if allowed is not None:
            g = int(allowed_row[r])
            lost = lost or g < -1 or g >= allowed.shape[0]
            if g >= 0 and not lost:
                for t in range(vocab):
                    if not (int(allowed[g, t // 32]) & 0xFFFFFFFF) >> (t % 32) & 1:
                        x[r, t] = -math.inf
        if lost:
            x[r, :] = -math.inf
    return x, steps * 2.0 ** -24 * np.where(np.isfinite(size), size, 0.0)


def truncated(logits, inv_temperature, top_k=0, top_p=1.0, min_p=0.0, u=0.0):
    """(token, tokens that stayed, log-probability) of one row."""
    x = np.asarray(logits, dtype=np.float64) + 0.0
    order = [i for i in np.argsort(np.where(np.isnan(x), np.inf, -x), kind="stable") if x[i] > -np.inf]
    if not order:
        return -1, 0, -math.inf
    if not inv_temperature > 0:
        return int(order[0]), 1, 0.0
    order = np.asarray(order)
    best = x[order[0]]
    if best == np.inf:
        return -1, 0, -math.inf
    if top_k > 0:
        order = order[:top_k]
    below = best - x[order]
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        w = np.where(below == 0, 1.0, np.exp(-np.where(below == 0, 0.0, below * float(inv_temperature))))
    if top_p < 1:
        mass = np.cumsum(w.astype(np.longdouble))
        n = 1
        while n < len(order) and mass[n - 1] < np.longdouble(top_p) * mass[-1]:
            n += 1
        order, w, below = order[:n], w[:n], below[:n]
    if min_p > 0:
        stays = (w >= min_p) | (below == 0)
        order, w = order[stays], w[stays]
    by_id = np.argsort(order)
    mass = np.cumsum(w[by_id].astype(np.longdouble))
    i = int(np.searchsorted(mass, np.longdouble(u) * mass[-1], side="right"))
    i = by_id[min(i, len(order) - 1)]
    return int(order[i]), len(order), float(np.log(w[i]) - np.log(mass[-1]))


def grow_tables(table, seats, held, lengths, page_size, pages):
    """(table, offsets)"""
    table, offsets = table.copy(), [0]
    for seat, have, n in zip(seats, held, lengths):
        blocks = -(-int(n) // page_size)
        need = max(0, blocks - int(have))
        if not 0 <= seat < table.shape[0] or have < 0 or blocks > table.shape[1]:
            need = 0
        if need and offsets[-1] + need <= len(pages):
            table[seat, have:have + need] = pages[offsets[-1]:offsets[-1] + need]
        offsets.append(offsets[-1] + need)
    return table, np.asarray(offsets, dtype=np.int32)


def step_rows(lengths, starts, seats, tables, page_size):
    """(q_start, positions, seats of the rows, slots per table)"""
    q_start, positions, tok_seat, slots = [0], [], [], [[] for _ in tables]
    for n, start, seat in zip(lengths, starts, seats):
        n = max(0, int(n))
        q_start.append(q_start[-1] + n)
        for x in range(int(start), int(start) + n):
            positions.append(x)
            tok_seat.append(int(seat))
            for table, out in zip(tables, slots):
                place = -1
                if 0 <= seat < table.shape[0] and 0 <= x // page_size < table.shape[1] and x >= 0:
                    page = int(table[seat, x // page_size])
                    place = page * page_size + x % page_size if page >= 0 else -1
                out.append(place if place < 1 << 31 else -1)
    return q_start, positions, tok_seat, slots
