"""Kernels that may begin before the one ahead of them has ended read their operands in a form that stays behind their wait.

A load that is marked as read-only (``__ldg``, ``ld.global.nc``, or through a ``const ... __restrict__`` parameter of a kernel) may be moved above
``wait_for_previous``, in front of the results that it is to read.  Checked in the sources: for every kernel that waits, its parameters, its
body and the bodies of the functions that it calls.
"""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "matterformer_b200" / "csrc"
READ_ONLY = re.compile(r"__ldg\s*\(|ld\.global(?:\.\w+)*\.nc\b|__ldca\s*\(|__ldcs\s*\(")


def _without_comments(text):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def _functions(text):
    """(name, what stands between the last statement and the body, body) of every function that the text defines."""
    found, i = [], 0
    for m in re.finditer(r"([A-Za-z_]\w*)\s*(?:<[^<>;(){}]*>)?\s*\(", text):
        if m.start() < i or m.group(1) in ("if", "for", "while", "switch", "sizeof", "decltype", "__launch_bounds__", "__maxnreg__", "__cluster_dims__"):
            continue
        at, depth = m.end(), 1
        while at < len(text) and depth:
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            at += 1
        end = re.match(r"\s*(?:const\s*)?\{", text[at:])
        if not end:
            continue
        head = text[max(text.rfind(";", 0, m.start()), text.rfind("}", 0, m.start())) + 1 : at]
        if "__device__" not in head and "__global__" not in head:
            continue
        body, depth, k = at + end.end(), 1, at + end.end()
        while k < len(text) and depth:
            depth += {"{": 1, "}": -1}.get(text[k], 0)
            k += 1
        found.append((m.group(1), head, text[body:k]))
        i = k
    return found


def _waiting_kernels():
    """(file, name, parameters, the bodies that run) of every kernel that waits for the kernel ahead of it."""
    headers = {p: _functions(_without_comments(p.read_text())) for p in CSRC.glob("*.cuh")}
    for path in sorted(CSRC.glob("*.cu*")):
        own = headers[path] if path in headers else _functions(_without_comments(path.read_text()))
        table = {}
        for name, head, body in [*own, *(f for p, fs in headers.items() if p != path for f in fs)]:
            if "__device__" in head:
                table.setdefault(name, []).append(body)
        for name, head, body in own:
            if "__global__" not in head or "wait_for_previous" not in body:
                continue
            seen, todo, bodies = set(), [body], []
            while todo:
                b = todo.pop()
                bodies.append(b)
                for callee in re.findall(r"([A-Za-z_]\w*)\s*(?:<[^;(){}]*>)?\s*\(", b):
                    if callee in table and callee not in seen:
                        seen.add(callee)
                        todo += table[callee]
                # members of the helpers' structs: v.load(...)
                for callee in re.findall(r"\.\s*([A-Za-z_]\w*)\s*\(", b):
                    if callee in table and callee not in seen:
                        seen.add(callee)
                        todo += table[callee]
            yield path.name, name, head, bodies


def test_the_kernels_are_found():
    names = {name for _, name, _, _ in _waiting_kernels()}
    assert {"gemm_kernel", "small_kernel", "rotary_kernel", "ln_modulate_bwd_kernel", "gated_residual_fwd_kernel", "column_sums_band_kernel",
            "block_list_kernel", "simplicial_rows_bwd_kernel", "band_fwd_kernel", "simplicial_small_res_fwd_kernel"} <= names  # fmt: skip
    launched = set()
    for path in CSRC.glob("*.cu"):
        launched |= set(re.findall(r"launch_dependent\(\s*(\w+_kernel)", path.read_text()))
    assert launched <= names, f"launched as dependents without a wait: {sorted(launched - names)}"


def test_no_operand_may_be_read_before_the_wait():
    wrong = []
    for file, name, head, bodies in _waiting_kernels():
        parameters = head[head.index(name) :]
        wrong += [f"{file}: {name}: {p.strip()}" for p in parameters.split(",") if "const" in p.split("*")[0] and "__restrict__" in p and "*" in p]
        wrong += [f"{file}: {name}: {m}" for b in bodies for m in READ_ONLY.findall(b)]
    assert not wrong, "\n".join(wrong)
