"""rope: HIP backend (hip_impl)."""
