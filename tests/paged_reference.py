"""Pages of a paged cache in plain Python: what dfattn_paged_fork, _free and _compact have to give."""

NONE = -1


def held(table, lens, page, n_pages, r, width=None):
    """(length, page ids) of row r."""
    width = len(table[r]) if width is None else width
    n = min(lens[r], width * page)
    return n, list(table[r][:-(-n // page)])


def count(rows, n_pages):
    refs = [0] * n_pages
    for ids in rows:
        for p in ids:
            if 0 <= p < n_pages:
                refs[p] += 1
    return refs


def by_use(refs):
    return [p for p, n in enumerate(refs) if n] + [p for p, n in enumerate(refs) if not n], sum(n > 0 for n in refs)


def fork(table, lens, parents, page, n_pages, keep=None):
    """dict of new rows (page ids), lens, refs, free_pages, free_start, copies [(src, dst)], cut."""
    rows, out_lens = [], []
    for i, r in enumerate(parents):
        if not 0 <= r < len(lens):
            rows.append([])
            out_lens.append(0)
            continue
        n, ids = held(table, lens, page, n_pages, r)
        if keep is not None:
            n = min(n, keep[i])
        rows.append(ids[:-(-n // page)])
        out_lens.append(n)
    refs = count(rows, n_pages)
    order, used = by_use(refs)
    writes = {}  # page -> children that will write behind their tokens in it, in order
    for i, n in enumerate(out_lens):
        if n % page and 0 <= rows[i][-1] < n_pages:
            writes.setdefault(rows[i][-1], []).append(i)
    full = {p: refs[p] - len(children) for p, children in writes.items()}
    copies, cut = [], 0
    for i, n in enumerate(out_lens):
        if not n % page or not 0 <= rows[i][-1] < n_pages:
            continue
        p = rows[i][-1]
        if writes[p][0] == i and not full[p]:
            continue
        refs[p] -= 1
        if used + len(copies) < n_pages:
            new = order[used + len(copies)]
            copies.append((p, new))
            rows[i][-1] = new
            refs[new] = 1
        else:
            cut += 1
            out_lens[i] = n // page * page
            # (the entry stays in the row, behind its tokens)
    return {"rows": rows, "lens": out_lens, "refs": refs, "free_pages": order, "free_start": used + len(copies),
            "copies": copies, "cut": cut}


def free(table, lens, page, n_pages, ended=None):
    lens = [0 if ended is not None and ended[r] else n for r, n in enumerate(lens)]
    refs = count([held(table, lens, page, n_pages, r)[1] for r in range(len(lens))], n_pages)
    order, used = by_use(refs)
    return {"lens": lens, "refs": refs, "free_pages": order, "free_start": used}


def compact(table, lens, page, n_pages):
    rows = [held(table, lens, page, n_pages, r)[1] for r in range(len(lens))]
    refs = count(rows, n_pages)
    used = sum(n > 0 for n in refs)
    src = [p for p in range(used, n_pages) if refs[p]]
    dst = [p for p in range(used) if not refs[p]]
    to = dict(zip(src, dst))
    new_refs = [0] * n_pages
    for p, n in enumerate(refs):
        new_refs[to.get(p, p)] += n
    return {"rows": [[to.get(p, p) for p in ids] for ids in rows], "refs": new_refs, "free_pages": list(range(n_pages)),
            "free_start": used, "copies": list(zip(src, dst))}
