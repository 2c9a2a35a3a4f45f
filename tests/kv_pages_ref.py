"""The pool of pages in plain Python: what kv_fork, kv_free and kv_compact leave, one item and one entry after the
other, from their description."""
import numpy as np

NONE = (-1, -1, 0, 0)


def pages_of(tokens, page):
    return -(-tokens // page)


def fork(refs, page, table, child_table, parent, child, length, capacity=None):
    """Updates refs and child_table; (copies, error bits)."""
    free = [p for p in range(len(refs)) if refs[p] == 0]
    copies, errors, taken = [], 0, 0
    rows, kids = len(table), len(child_table)
    table = table.copy()
    for i in range(len(child)):
        copies.append(NONE)
        if child[i] < 0:
            continue
        n = int(length[i])
        room = n if capacity is None else max(n, int(capacity[i]))
        end, held = pages_of(room, page), pages_of(max(n, 0), page)
        if child[i] >= kids or not -1 <= parent[i] < rows or n < 0 or room > 1 << 30 or end > child_table.shape[1] or (
                parent[i] >= 0 and held > table.shape[1]):
            errors |= 8
            continue
        first, part = held, 0
        if parent[i] >= 0:
            first, part = n // page, n % page
            for j in range(first):
                p = int(table[parent[i], j])
                if 0 <= p < len(refs):
                    refs[p] += 1
                else:
                    p, errors = -1, errors | 1
                child_table[child[i], j] = p
        for j in range(first, end):
            p = free[taken] if taken < len(free) else -1
            taken += 1
            child_table[child[i], j] = p
            if p < 0:
                errors |= 16
                continue
            refs[p] = 1
            if part and j == first:
                src = int(table[parent[i], j])
                if 0 <= src < len(refs):
                    copies[-1] = (src, p, part, 0)
                else:
                    errors |= 1
    return np.array(copies, np.int32).reshape(-1, 4), errors


def free(refs, page, table, row, length):
    errors = 0
    for r, n in zip(row, length):
        if r < 0:
            continue
        if r >= len(table) or n < 0 or pages_of(n, page) > table.shape[1]:
            errors |= 8
            continue
        for p in table[r, :pages_of(n, page)]:
            if p < 0:
                continue
            if p >= len(refs):
                errors |= 1
            elif refs[p] <= 0:
                errors |= 32
            else:
                refs[p] -= 1
    return errors


def compact(refs, page, table, new_table, length):
    """(new refs, page map, copies, error bits); fills new_table."""
    used = int((refs != 0).sum())
    where = {p: p for p in range(len(refs)) if refs[p] and p < used}
    src = [p for p in range(used, len(refs)) if refs[p]]
    dst = [p for p in range(used) if not refs[p]]
    where.update(zip(src, dst))
    new = np.zeros_like(refs)
    for p, q in where.items():
        new[q] = refs[p]
    errors = 0
    table = table.copy()
    for b, n in enumerate(length):
        if n < 0 or pages_of(n, page) > min(table.shape[1], new_table.shape[1]):
            errors |= 8
            continue
        for j in range(pages_of(n, page)):
            p = int(table[b, j])
            new_table[b, j] = where.get(p, -1)
            if p != -1 and p not in where:
                errors |= 1
    page_map = np.array([where.get(p, -1) for p in range(len(refs))], np.int32)
    return new, page_map, np.array([(a, b, page, 0) for a, b in zip(src, dst)], np.int32).reshape(-1, 4), errors
