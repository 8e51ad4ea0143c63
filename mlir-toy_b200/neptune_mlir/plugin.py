"""Helpers for locating native libraries.

``find_library_path`` resolves the nb200 kernel library the same way the reference resolves its
dialect plugin: explicit argument, then an environment variable, then the installed package
directory, then common build directories.  The resolution code (``_find_in_dir``, ``_candidate_dirs``
and the loop in ``_resolve``) is adapted from the reference's src/neptune_mlir/plugin.py:10-55,
generalised from one library to three; the interface is one this build keeps on purpose.  ``find_plugin_path`` keeps the
reference's name and contract for the HTile dialect plugin; this build reads HTile text itself and
never needs that plugin, so the function usually returns None.
"""

import os
from pathlib import Path

DEFAULT_PLUGIN_ENV = "NEPTUNE_MLIR_PLUGIN"
PLUGIN_PATTERNS = ("libHTileDialectPlugin.*",)
DEFAULT_LIBRARY_ENV = "NEPTUNE_B200_LIB"
LIBRARY_PATTERNS = ("libnb200.so", "libnb200.*")
DEFAULT_FRONT_ENV = "NEPTUNE_HTILE_FRONT_LIB"
BINDING_PATTERNS = ("nb200_torch.so", "nb200_torch.*")
FRONT_PATTERNS = ("libhtile_front.so", "libhtile_front.*")


def _find_in_dir(directory: Path, patterns) -> Path | None:
    for pattern in patterns:
        matches = sorted(directory.glob(pattern))
        if matches:
            return matches[0]
    return None


def _candidate_dirs() -> list[Path]:
    pkg_dir = Path(__file__).resolve().parent
    repo_root = pkg_dir.parents[1] if len(pkg_dir.parents) >= 2 else pkg_dir
    return [
        pkg_dir / "_native",
        repo_root / "build",
        Path.cwd() / "build",
    ]


def _resolve(explicit, env_name: str, patterns) -> Path | None:
    candidates: list[Path] = []
    if explicit:
        candidates.append(Path(explicit).expanduser())
    env_path = os.environ.get(env_name)
    if env_path:
        candidates.append(Path(env_path).expanduser())
    for candidate in candidates:
        if candidate.is_file():
            return candidate.resolve()
    for directory in _candidate_dirs():
        if not directory.is_dir():
            continue
        if (match := _find_in_dir(directory, patterns)) is not None:
            return match.resolve()
    return None


def find_library_path(explicit: str | os.PathLike[str] | None = None) -> Path | None:
    """Resolve libnb200.so: explicit path, $NEPTUNE_B200_LIB, neptune_mlir/_native, <repo>/build, <cwd>/build."""
    return _resolve(explicit, DEFAULT_LIBRARY_ENV, LIBRARY_PATTERNS)


def find_front_path(explicit: str | os.PathLike[str] | None = None) -> Path | None:
    """Resolve libhtile_front.so (the C++ HTile front end), same search order with $NEPTUNE_HTILE_FRONT_LIB."""
    return _resolve(explicit, DEFAULT_FRONT_ENV, FRONT_PATTERNS)


def find_binding_path(library: Path | None = None) -> Path | None:
    """Resolve nb200_torch.so (the CPython module between torch tensors and the kernel library): beside ``library``, the
    kernel library that was loaded, then in the same directories."""
    directories = [*([library.parent] if library else []), *_candidate_dirs()]
    return next((m.resolve() for d in directories if d.is_dir() and (m := _find_in_dir(d, BINDING_PATTERNS))), None)


def find_plugin_path(explicit: str | os.PathLike[str] | None = None) -> Path | None:
    """Resolve the HTile dialect plugin path (same order as the reference's function of this name)."""
    return _resolve(explicit, DEFAULT_PLUGIN_ENV, PLUGIN_PATTERNS)
