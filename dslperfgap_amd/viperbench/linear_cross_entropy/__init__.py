"""linear_cross_entropy: HIP backend (hip_impl)."""
